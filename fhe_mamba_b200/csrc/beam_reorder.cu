// Reordering of states after a selection (fhe_beam_reorder): row i of each batch
// item's beams becomes its row parents[i], in place, for every tensor at once.
//
// A thread owns the same 16 bytes of all of an item's rows, and the next 16 of the
// block's after them: it brings the rows that others take into its own part of shared
// memory by asynchronous copies, up to three steps ahead, waits for them, and then
// writes the rows that change.  So no thread reads what another writes, nothing waits
// for another thread, and only rows that change are written, only their parents read.
// Memory bounds it.
#include <algorithm>

#include "launch_count.h"
#include "mamba_ops.h"

namespace fhe {
namespace {

constexpr uint32_t kMaxBeams = 64, kTable = 64, kThreads = 128, kStep = kThreads * 16;  // bytes of a row in a step
// Rows' steps in shared memory, as many as beams where those are more.  More of them
// ahead scatter the traffic: 16 x 8 beams of 24 layers, three rows of eight moved, 1.84 GB
// read and written: 287 us with 8 (98% of a copy's rate), 328 us with 16.
constexpr uint32_t kSlots = 8;

struct State {
  uint8_t* p;
  uint64_t row;    // bytes
  uint32_t first;  // block of the grid
  uint32_t word;   // bytes that rows and base are multiples of, up to 16
};
struct ReorderArgs {
  State state[kTable];
  uint32_t n, beams, steps;  // steps of a block
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

// The block's steps from byte `at` of each row, as words of type W, D - 1 steps ahead.
template <class W, int D>
__device__ __forceinline__ void move(uint8_t* base, uint64_t row, uint64_t at, uint32_t steps, const uint8_t* parent,
                                     uint64_t wanted, uint64_t changed, uint8_t* shared) {
  constexpr int N = 16 / sizeof(W);
  const uint32_t tid = threadIdx.x, each_step = __popcll(wanted);
  auto each = [&](uint64_t rows, auto&& f) {
    for (; rows; rows &= rows - 1) f((uint32_t)__ffsll((long long)rows) - 1);
  };
  auto here = [&](uint32_t step, uint32_t slot, int i) {
    return reinterpret_cast<W*>(shared + (step % D * each_step + slot) * kStep) + i * kThreads + tid;
  };
  auto there = [&](uint32_t step, int i) { return at + step * kStep + (i * kThreads + tid) * sizeof(W); };
  auto fetch = [&](uint32_t step) {
    uint32_t slot = 0;
    if (step < steps)
      each(wanted, [&](uint32_t r) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (there(step, i) < row) bring(here(step, slot, i), reinterpret_cast<const W*>(base + r * row + there(step, i)));
        ++slot;
      });
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < D - 1; ++i) fetch(i);
  for (uint32_t step = 0; step < steps && at + step * kStep < row; ++step) {
    fetch(step + D - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
    each(changed, [&](uint32_t r) {
      const uint32_t from = __popcll(wanted & ((1ull << parent[r]) - 1));
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (there(step, i) < row) *reinterpret_cast<W*>(base + r * row + there(step, i)) = *here(step, from, i);
    });
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

__global__ void __launch_bounds__(kThreads) k_reorder(const __grid_constant__ ReorderArgs g) {
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
  const uint64_t at = (uint64_t)(blockIdx.x - s.first) * g.steps * kStep;
  uint8_t* base = s.p + (uint64_t)item * K * s.row;
  const uint32_t n = __popcll(wanted), slots = max(K, kSlots);
  auto with = [&](auto w) {
    using W = decltype(w);
    if (n * 4 <= slots) move<W, 4>(base, s.row, at, g.steps, parent, wanted, changed, shared);
    else if (n * 2 <= slots) move<W, 2>(base, s.row, at, g.steps, parent, wanted, changed, shared);
    else move<W, 1>(base, s.row, at, g.steps, parent, wanted, changed, shared);
  };
  if (s.word == 16) with(uint4{});
  else if (s.word == 8) with(uint2{});
  else if (s.word == 4) with(uint32_t{});
  else if (s.word == 2) with(uint16_t{});
  else with(uint8_t{});
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
  const uint32_t shared = std::max(a.beams, kSlots) * kStep;
  if (shared > 32768) allow_shared(k_reorder, kMaxBeams * kStep);
  // up to 16 steps to a block, fewer where that leaves places on the SMs empty
  uint64_t all = 0;
  for (uint32_t i = 0; i < a.count; ++i) all += (a.row_bytes[i] + kStep - 1) / kStep;
  uint32_t steps = 16;
  while (steps > 1 && all * a.batch / steps < 148 * 14) steps /= 2;
  for (uint32_t i = 0; i < a.count;) {
    ReorderArgs g{};
    g.beams = a.beams;
    g.steps = steps;
    g.parents = a.parents;
    uint64_t blocks = 0;
    for (; i < a.count && g.n < kTable; ++i) {
      const uint64_t row = a.row_bytes[i];
      if (row == 0) continue;
      const uint64_t more = (row + steps * kStep - 1) / (steps * kStep);
      if (blocks + more >= (1ull << 31)) break;
      const uint64_t bits = row | reinterpret_cast<uintptr_t>(a.states[i]) | 16;
      g.state[g.n++] = State{static_cast<uint8_t*>(a.states[i]), row, (uint32_t)blocks, (uint32_t)(bits & (0 - bits))};
      blocks += more;
    }
    if (g.n == 0) continue;
    k_reorder<<<dim3((uint32_t)blocks, a.batch), kThreads, shared, static_cast<cudaStream_t>(a.stream)>>>(g);
    note_launch();
    FHE_CUDA(cudaGetLastError());
  }
}

}  // namespace fhe
