// Gradients of the root-mean-square norms (fhe_rms_norm_backward).
//
// With a = dy w and u = h r: dh = r (a - u mean(a u)) (+ the gradient that h
// itself has), dweight = sum over rows of dy u.  Like the norm, a row is spread
// over one to sixteen warps and read once.  Its words come by asynchronous copies
// through each thread's own part of shared memory, rows ahead, and are taken from
// there twice, for the mean and for the gradients; pairs and single elements are held
// in registers.  Two chunks of them fit; groups of more than 8192 channels that are not
// loaded as words, or whose row is too large for the ring (float32 with a factor for each
// of 16384 channels), take four, much of which the compiler spills to local memory (norm
// and gradients of 2000 x 12290 bfloat16 on float32: 0.38 ms, of 2000 x 16384 float32
// with factors 0.81 ms, a quarter of a copy's rate).  A block keeps its share of the sums
// over rows in registers from row to row, and a second launch (4 to 6 us) adds the
// blocks' shares in a fixed order.
// 32768 rows of 768, bfloat16 and a float32 stream: 70 us, 5.8 TB/s; 32768 x 1536
// bfloat16 with a gate: 81 us, 6.2 TB/s.
#include "launch_count.h"
#include "norms.h"

namespace fhe {
namespace {

// A lane's words of a row in the ring: h or x, dy, gate or (for the channel scale) x,
// dh.  What is read twice stays out of the registers, and the loads of the next rows
// run behind the arithmetic of this one.
template <int MODE, class A, class H, int N>
struct GradWords {
  using S = std::conditional_t<MODE == kNormGate, A, H>;
  static constexpr bool kAdd = MODE == kNormAdd || MODE == kNormAddScaled, kThird = MODE == kNormGate || MODE == kNormAddScaled;
  static constexpr int kS = 0, kDy = kS + N * Eight<S>::kQuads, kZ = kDy + N * Eight<A>::kQuads,
                       kDh = kZ + (kThird ? N * Eight<A>::kQuads : 0), kAll = kDh + (kAdd ? N * Eight<H>::kQuads : 0);
};

template <int MODE, class A, class H, int N, int LAY>
__global__ void __launch_bounds__(N == 3 ? 256 : 512) k_norm_grad(const NormArgs g) {
  __shared__ float red[2][16];
  extern __shared__ __align__(16) float sums[];  // the ring of rows; then sums over a block's rows
  constexpr bool kNarrow = is_narrow(LAY), kRing = LAY == kWords;  // words of wide rows come through the ring
  RowSum<kNarrow> row_sum{red, g.lanes};
  using W = GradWords<MODE, A, H, N>;
  constexpr bool kAdd = W::kAdd, kScaled = MODE == kNormAddScaled, kThird = W::kThird;
  using X = std::conditional_t<MODE == kNormPlain, H, A>;  // x
  using S = typename W::S;                                 // what h is made from
  const uint32_t c0 = blockIdx.y * g.gw + from<N, LAY>(g.lanes);
  const int left = (int)g.gw - (int)from<N, LAY>(g.lanes);
  Eight<float> w[N], cs[kScaled ? N : 1];
  float dw[N][8], dcs[kScaled ? N : 1][8];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    w[c].clear();
    load_chunk<LAY>(w[c], g.weight + c0, c, left);
    vset(dw[c], 0.f);
    if constexpr (kScaled) {
      cs[c].clear();
      load_chunk<LAY>(cs[c], g.cscale + c0, c, left);
      vset(dcs[c], 0.f);
    }
  }
  const float n = 1.f / (float)g.gw;
  const Ring<W::kAll> ring(sums, g.stages);
  Eight<S> s[kRing ? 1 : N];
  Eight<A> dy[kRing ? 1 : N], z[kThird && !kRing ? N : 1];
  Eight<H> dh[kAdd && !kRing ? N : 1];
  // a warp's first row, and this lane's among its rows
  const uint32_t rows = kNarrow ? 32 / g.lanes : 1, sub = kNarrow ? threadIdx.x / g.lanes : 0;
  const uint32_t step = gridDim.x * blockDim.y * rows, base0 = (blockIdx.x * blockDim.y + threadIdx.y) * rows;
  int stage = 0;
  auto fetch = [&](uint32_t row, [[maybe_unused]] int to) {
    if (row < g.rows) {
      const int64_t out = (int64_t)row * g.width + c0;
      const S* sp = kAdd ? static_cast<const S*>(g.h) + out : static_cast<const S*>(g.x) + (int64_t)row * g.xs + c0;
      const A* dyp = static_cast<const A*>(g.dy) + out;
      const A* zp = MODE == kNormGate ? static_cast<const A*>(g.gate) + (int64_t)row * g.gs + c0
                                      : static_cast<const A*>(g.x) + (int64_t)row * g.xs + c0;
      const H* dhp = static_cast<const H*>(g.dh) + out;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if constexpr (kRing) {
          ring.copy(to, W::kS, sp, c, left);
          ring.copy(to, W::kDy, dyp, c, left);
          if constexpr (kThird) ring.copy(to, W::kZ, zp, c, left);
          if constexpr (kAdd)
            if (g.dh) ring.copy(to, W::kDh, dhp, c, left);
        } else {
          load_chunk<LAY>(s[c], sp, c, left);
          load_chunk<LAY>(dy[c], dyp, c, left);
          if constexpr (kThird) load_chunk<LAY>(z[c], zp, c, left);
          if constexpr (kAdd)
            if (g.dh) load_chunk<LAY>(dh[c], dhp, c, left);
        }
      }
    }
    if constexpr (kRing) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // chunk c of an array, from the ring or the registers; 0 past the row's end
  auto take = [&](auto& held, int first, int c, float (&o)[8]) {
    if constexpr (kRing) {
      std::remove_reference_t<decltype(held[0])> e;
      ring.take(e, stage, first, c);
      e.floats(o);
    } else {
      held[c].floats(o);
    }
  };
  if constexpr (kRing) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      ring.blank(g.stages, W::kS, (const S*)nullptr, c, left);
      ring.blank(g.stages, W::kDy, (const A*)nullptr, c, left);
      if constexpr (kThird) ring.blank(g.stages, W::kZ, (const A*)nullptr, c, left);
      if constexpr (kAdd) ring.blank(g.stages, W::kDh, (const H*)nullptr, c, left);
    }
    for (int i = 0; i + 1 < g.stages; ++i) fetch(base0 + i * step, i);
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      s[c].clear();
      dy[c].clear();
      if constexpr (kThird) z[c].clear();
      if constexpr (kAdd) dh[c].clear();
    }
  }
  for (uint32_t base = base0; base < g.rows; base += step) {
    const uint32_t row = base + sub;
    const bool live = !kNarrow || row < g.rows;
    const int64_t out = (int64_t)row * g.width + c0;
    const float r = live ? g.rstd[(int64_t)row * g.groups + blockIdx.y] : 0.f;
    if constexpr (kRing) {
      __syncwarp();  // the row to be filled has been read
      fetch(row + (g.stages - 1) * step, stage ? stage - 1 : g.stages - 1);
      wait_copies(g.stages);
    } else {
      fetch(row, 0);
    }
    float rr[8];
    vset(rr, r);
    // u = h r; with a gate also p = SiLU(gate), from its sigmoid, which is kept
    float q[MODE == kNormGate ? N : 1][8];
    auto unit = [&](int c, bool first, float (&u)[8], float (&xf)[8], float (&p)[8]) {
      take(s, W::kS, c, xf);
      if constexpr (MODE == kNormGate) {
        float zf[8];
        take(z, W::kZ, c, zf);
        if (first) gate_sigmoid<A>(q[c], zf);
        vmul(p, q[c], zf);
        vmul(u, xf, p);
        vmul(u, u, rr);
      } else {
        vmul(u, xf, rr);
      }
    };
    if constexpr (kNarrow) {
      if (!live) {  // rows past the last add nothing
        s[0].clear();
        dy[0].clear();
        if constexpr (kThird) z[0].clear();
      }
    }
    float part[2][2] = {};
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float u[8], xf[8], p[8], d[8], wf[8];
      unit(c, true, u, xf, p);
      take(dy, W::kDy, c, d);
      w[c].floats(wf);
      vmul(d, d, u);
      vadd(dw[c], dw[c], d);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float aa[2] = {d[i], d[i + 1]}, ww[2] = {wf[i], wf[i + 1]};
        vfma(part[i / 2 % 2], aa, ww, part[i / 2 % 2]);
      }
    }
    const float m = row_sum((part[0][0] + part[0][1]) + (part[1][0] + part[1][1])) * n;
    if (!live) continue;
    float mm[8];
    vset(mm, -m);
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float u[8], xf[8], p[8], d[8], wf[8];
      unit(c, false, u, xf, p);
      take(dy, W::kDy, c, d);
      w[c].floats(wf);
      vmul(d, d, wf);
      vfma(d, u, mm, d);
      if constexpr (kAdd) {
        float e[8];
        vset(e, 0.f);
        if (g.dh) take(dh, W::kDh, c, e);
        vfma(d, d, rr, e);
      } else {
        vmul(d, d, rr);
      }
      if constexpr (MODE == kNormGate) {
        float o[8], one[8];
        Eight<A> e;
        vmul(o, d, p);
        e.set(o);
        if (g.dx) store_chunk<LAY>(e, static_cast<A*>(g.dx) + out, c, left);
        // SiLU' = q (1 + z (1 - q)) = q + p (1 - q)
#pragma unroll
        for (int i = 0; i < 8; ++i) one[i] = 1.f - q[c][i];
        vfma(o, p, one, q[c]);
        vmul(d, d, xf);
        vmul(o, o, d);
        e.set(o);
        if (g.dgate) store_chunk<LAY>(e, static_cast<A*>(g.dgate) + out, c, left);
      } else {
        if constexpr (kScaled) {
          float xg[8];
          take(z, W::kZ, c, xg);
          vfma(dcs[c], d, xg, dcs[c]);
        }
        if constexpr (kAdd) {
          Eight<H> e;
          e.set(d);
          if (g.dres) store_chunk<LAY>(e, static_cast<H*>(g.dres) + out, c, left);
          float sc[8];
          vset(sc, g.scale);
          vmul(d, d, sc);
          if constexpr (kScaled) {
            cs[c].floats(sc);
            vmul(d, d, sc);
          }
        }
        Eight<X> e;
        e.set(d);
        if (g.dx) store_chunk<LAY>(e, static_cast<X*>(g.dx) + out, c, left);
      }
    }
    stage = stage + 1 == g.stages ? 0 : stage + 1;
  }
  if constexpr (kRing) asm volatile("cp.async.wait_all;" ::: "memory");
  if constexpr (kNarrow) {  // the warp's rows together
    for (uint32_t o = g.lanes; o < 32; o *= 2)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[0][i] += __shfl_xor_sync(~0u, dw[0][i], o);
        if constexpr (kScaled) dcs[0][i] += __shfl_xor_sync(~0u, dcs[0][i], o);
      }
  }
  // the block's rows together, one after the other
  auto gather = [&](float (&v)[N][8], float* to, float k) {
    float* sum = sums + from<N, LAY>(g.lanes);
    for (uint32_t turn = 0; turn < blockDim.y; ++turn) {
      __syncthreads();
      if (threadIdx.y != turn) continue;
#pragma unroll
      for (int c = 0; c < N; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = away<LAY>(c, i);
          if (at >= left || (kNarrow && sub != 0)) continue;
          const float all = turn ? sum[at] + v[c][i] : v[c][i];
          if (turn + 1 == blockDim.y) to[at] = all * k;
          else sum[at] = all;
        }
    }
  };
  if (g.part) {
    float* to = g.part + (int64_t)blockIdx.x * g.width + c0;
    gather(dw, to, 1.f);
    if constexpr (kScaled) gather(dcs, to + (int64_t)gridDim.x * g.width, g.scale);
  }
}

// Adds the blocks' shares: 32 channels x 32 strands of blocks.
__global__ void __launch_bounds__(1024) k_norm_sum(const float* part, uint32_t blocks, uint32_t width, float* dweight,
                                                   float* dcscale) {
  __shared__ float s[32][33];
  const uint32_t c = blockIdx.x * 32 + threadIdx.x;
  float* out = blockIdx.y ? dcscale : dweight;
  if (!out) return;
  part += (int64_t)blockIdx.y * blocks * width;
  float v = 0.f;
  if (c < width) {
#pragma unroll 10
    for (uint32_t b = threadIdx.y; b < blocks; b += 32) v += part[(int64_t)b * width + c];
  }
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = s[threadIdx.x][threadIdx.y];  // strand x of channel y
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < width) out[blockIdx.x * 32 + threadIdx.y] = v;
}

uint32_t together(const fhe_rms_norm_grad_args& a) {
  const fhe_rms_norm_args& f = a.f;
  const uint32_t ea = elem_size(f.dtype), eh = f.gate ? ea : elem_size(f.stream_dtype);
  const uint32_t ex = f.gate || f.residual ? ea : eh;
  Together t(f.width / f.groups);
  if (!f.residual || f.channel_scale) t.with(f.x, f.x_stride, ex);
  if (f.residual) t.with(f.h, f.width, eh);
  if (f.gate) t.with(f.gate, f.gate_stride, ea);
  t.with(f.channel_scale, 0, 4);
  t.with(f.weight, 0, 4);
  t.with(a.dy, f.width, ea);
  t.with(a.dh, f.width, eh);
  t.with(a.dx, f.width, ex);
  t.with(a.dresidual, f.width, eh);
  t.with(a.dgate, f.width, ea);
  return t.n;
}

// How a call is laid out: shape, rows of the ring, shared memory, and blocks that go
// from row to row, as many as are resident.
struct GradPlan {
  NormShape shape;
  uint32_t together, stages, shared, blocks;
};
GradPlan grad_plan(const fhe_rms_norm_grad_args& a, uint32_t together) {
  const fhe_rms_norm_args& f = a.f;
  const uint32_t gw = f.width / f.groups;
  const uint32_t wa = elem_size(f.dtype) / 2, wh = f.gate ? wa : elem_size(f.stream_dtype) / 2;
  const uint32_t per_chunk = (f.gate ? wa : wh) + wa + (f.gate || f.channel_scale ? wa : 0) + (f.residual ? wh : 0);
  GradPlan p{};
  p.together = together;
  for (;; p.together = 2) {
    p.shape = norm_shape(gw, (uint64_t)f.rows * f.groups, p.together, f.gate != nullptr);
    const uint32_t warps = p.shape.warps == 1 ? 4 : p.shape.warps;  // of a block
    uint32_t resident = std::max(1u, 16 / warps);
    p.shared = p.shape.warps == 1 ? gw * sizeof(float) : 0;  // one warp's channels, at most 1024
    if (p.shape.layout(p.together) == kWords) {
      const uint32_t row = p.shape.chunks * per_chunk * 16 * 32 * warps;
      if (row + kBlockShared > kSmShared) continue;
      const RingPlan r = ring_plan(row, warps, 120 * 1024);
      p.stages = r.stages;
      p.shared = std::max(p.shared, p.stages * row);
      resident = r.blocks;
    }
    p.blocks = std::max(1u, std::min((f.rows + p.shape.rows_per_block - 1) / p.shape.rows_per_block,
                                     std::max(1u, 148 * resident / f.groups)));
    return p;
  }
}

bool sums_wanted(const fhe_rms_norm_grad_args& a) { return a.dweight || a.dchannel_scale; }

}  // namespace

uint64_t rms_norm_backward_workspace(const fhe_rms_norm_grad_args& a) {
  check_norm(a.f);
  if (!sums_wanted(a)) return 0;
  // enough for these sizes wherever the arrays lie: the workspace may be asked for before they exist
  const uint32_t most = Together(a.f.width / a.f.groups).n;
  uint32_t blocks = 0;
  for (uint32_t n : {1u, 2u, 8u})
    if (n <= most) blocks = std::max(blocks, grad_plan(a, n).blocks);
  return (uint64_t)blocks * a.f.width * sizeof(float) * (a.f.channel_scale ? 2 : 1);
}

void rms_norm_backward(const fhe_rms_norm_grad_args& a) {
  check_norm(a.f);
  const fhe_rms_norm_args& f = a.f;
  require(f.rows == 0 || (f.weight && f.rstd && a.dy && (f.residual ? f.h != nullptr : f.x != nullptr)), "null input");
  require(f.rows == 0 || !f.channel_scale || f.x, "null input");
  require(!a.dgate || f.gate, "dgate without a gate");
  require((!a.dresidual && !a.dh) || f.residual, "dresidual or dh without a residual");
  require(!a.dchannel_scale || f.channel_scale, "dchannel_scale without a channel_scale");
  check_workspace(a.workspace, a.workspace_bytes, rms_norm_backward_workspace(a));
  DeviceGuard dev(f.device);
  cudaStream_t st = static_cast<cudaStream_t>(a.stream);
  if (f.rows == 0) {
    if (a.dweight) FHE_CUDA(cudaMemsetAsync(a.dweight, 0, (size_t)f.width * 4, st));
    if (a.dchannel_scale) FHE_CUDA(cudaMemsetAsync(a.dchannel_scale, 0, (size_t)f.width * 4, st));
    return;
  }
  NormArgs g = norm_args(f);
  g.dy = a.dy;
  g.dh = a.dh;
  g.dx = a.dx;
  g.dres = a.dresidual;
  g.dgate = a.dgate;
  g.part = sums_wanted(a) ? static_cast<float*>(a.workspace) : nullptr;
  const GradPlan p = grad_plan(a, together(a));
  g.stages = (int)p.stages;
  g.lanes = p.shape.lanes;
  with_norm(f, p.shape.chunks, p.shape.layout(p.together), [&](auto mode, auto act, auto str, auto chunks, auto layout) {
    auto k = k_norm_grad<decltype(mode)::value, decltype(act), decltype(str), decltype(chunks)::value,
                         decltype(layout)::value>;
    if (p.shared > 48000) allow_shared(k, kSmShared - kBlockShared);
    const dim3 block(32 * p.shape.warps, p.shape.warps == 1 ? 4 : 1);
    k<<<dim3(p.blocks, f.groups), block, p.shared, st>>>(g);
  });
  note_launch();
  if (g.part) {
    k_norm_sum<<<dim3((f.width + 31) / 32, f.channel_scale ? 2 : 1), dim3(32, 32), 0, st>>>(
        g.part, p.blocks, f.width, a.dweight, a.dchannel_scale);
    note_launch();
  }
  FHE_CUDA(cudaGetLastError());
}

}  // namespace fhe
