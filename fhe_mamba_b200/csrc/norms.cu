// Root-mean-square norms with their residual or their gate (fhe_rms_norm).
//
// y = h r w with r = 1 / sqrt(mean(h^2) + eps) over a row, or over each group of a
// row, of h = x, residual + scale x (stored in the stream's type, which is what
// the norm is of) or x SiLU(gate).  A row lies in the registers of one to sixteen
// warps, eight channels to a 16-byte word, so its inputs are read once and its
// outputs written once: memory bounds it.  The weights stay in registers while a
// block goes from row to row.  32768 rows of 768, bfloat16 added to a float32 stream: 47
// us, 6.4 TB/s (97% of a measured copy); 32768 x 1536 bfloat16 with a gate out of rows of
// 3352: 49 us, 6.2 TB/s; 4 rows: 1.9 us.
#include "launch_count.h"
#include "norms.h"

namespace fhe {
namespace {

template <int MODE, class A, class H, int N, int LAY>
__global__ void __launch_bounds__(512) k_norm(const NormArgs g) {
  __shared__ float red[2][16];
  extern __shared__ __align__(16) uint8_t shared[];
  constexpr bool kNarrow = is_narrow(LAY);
  RowSum<kNarrow> row_sum{red, g.lanes};
  constexpr bool kTwo = MODE != kNormPlain, kRing = MODE == kNormGate && LAY == kWords;
  using X = std::conditional_t<MODE == kNormPlain, H, A>;
  using Y = std::conditional_t<MODE == kNormGate, A, H>;  // gate or residual
  const uint32_t c0 = blockIdx.y * g.gw + from<N, LAY>(g.lanes);
  const int left = (int)g.gw - (int)from<N, LAY>(g.lanes);
  const X* xp = static_cast<const X*>(g.x) + c0;
  const Y* yp = static_cast<const Y*>(MODE == kNormGate ? g.gate : g.res) + c0;
  const int64_t ys = MODE == kNormGate ? g.gs : g.rs;
  Eight<float> w[N], cs[MODE == kNormAddScaled ? N : 1];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    w[c].clear();
    load_chunk<LAY>(w[c], g.weight + c0, c, left);
    if constexpr (MODE == kNormAddScaled) {
      cs[c].clear();
      load_chunk<LAY>(cs[c], g.cscale + c0, c, left);
    }
  }
  const float n = 1.f / (float)g.gw;
  // a warp's first row, and this lane's among its rows
  const uint32_t rows = kNarrow ? 32 / g.lanes : 1, sub = kNarrow ? threadIdx.x / g.lanes : 0;
  const uint32_t step = gridDim.x * blockDim.y * rows;
  uint32_t base = (blockIdx.x * blockDim.y + threadIdx.y) * rows;
  // The next row's words come while this one is summed and written: into registers,
  // or with a gate, whose sigmoids take longer, a row ahead through a ring (32768 x 1536
  // bfloat16: 50 us, 65 with loads in registers).
  Eight<X> e[N];
  Eight<Y> f[kTwo ? N : 1];
  constexpr int kQ = Eight<A>::kQuads;
  const Ring<2 * N * kQ> ring(shared, g.stages);
  int stage = 0;
  auto fetch = [&](uint32_t at, [[maybe_unused]] int to) {
    if (at < g.rows) {
      const X* x = xp + (int64_t)at * g.xs;
      const Y* y = yp + (int64_t)at * ys;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        if constexpr (kRing) {
          ring.copy(to, 0, x, c, left);
          ring.copy(to, N * kQ, y, c, left);
        } else {
          load_chunk<LAY>(e[c], x, c, left);
          if constexpr (kTwo) load_chunk<LAY>(f[c], y, c, left);
        }
      }
    }
    if constexpr (kRing) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (kRing) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      ring.blank(g.stages, 0, xp, c, left);
      ring.blank(g.stages, N * kQ, yp, c, left);
    }
    for (int i = 0; i + 1 < g.stages; ++i) fetch(base + i * step, i);
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      e[c].clear();
      if constexpr (kTwo) f[c].clear();
    }
    fetch(base + sub, 0);
  }
  for (; base < g.rows; base += step) {
    const uint32_t row = base + sub;
    const bool live = !kNarrow || row < g.rows;
    if constexpr (kRing) {
      __syncwarp();  // the row to be filled has been read
      fetch(row + (g.stages - 1) * step, stage ? stage - 1 : g.stages - 1);
      wait_copies(g.stages);
#pragma unroll
      for (int c = 0; c < N; ++c) {
        ring.take(e[c], stage, 0, c);
        ring.take(f[c], stage, N * kQ, c);
      }
      stage = stage + 1 == g.stages ? 0 : stage + 1;
    }
    float h[N][8];
    [[maybe_unused]] H* out = static_cast<H*>(g.h) + (int64_t)row * g.width + c0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      e[c].floats(h[c]);
      if constexpr (MODE == kNormGate) {
        float q[8], zf[8];
        f[c].floats(zf);
        gate_sigmoid<A>(q, zf);
        vmul(q, q, zf);
        vmul(h[c], h[c], q);
      } else if constexpr (kTwo) {
        float rf[8], s[8];
        f[c].floats(rf);
        vset(s, g.scale);
        if constexpr (MODE == kNormAddScaled) {
          float v[8];
          cs[c].floats(v);
          vmul(s, s, v);
        }
        vfma(h[c], s, h[c], rf);
        Eight<H> kept;
        kept.set(h[c]);
        if (live) store_chunk<LAY>(kept, out, c, left);
        kept.floats(h[c]);
      }
    }
    if constexpr (!kRing) fetch(row + step, 0);
    float part[2][2] = {};
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float p[2] = {h[c][i], h[c][i + 1]};
        vfma(part[i / 2 % 2], p, p, part[i / 2 % 2]);
      }
    const float ss = row_sum((part[0][0] + part[0][1]) + (part[1][0] + part[1][1]));
    float r = rsqrtf(fmaf(ss, n, g.eps));
    // squares past fp32's range: the row again, scaled (an infinity of the row itself gives r = 0)
    if (kNarrow ? __any_sync(~0u, ss == INFINITY) : ss == INFINITY) {
      const float k = 0x1p-80f;
      float again = 0.f;
#pragma unroll
      for (int c = 0; c < N; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) again = fmaf(h[c][i] * k, h[c][i] * k, again);
      again = row_sum(again);
      if (ss == INFINITY) r = k / sqrtf(again * n);
    }
    if (!live) continue;
    if (g.rstd && (kNarrow ? threadIdx.x % g.lanes : threadIdx.x) == 0) g.rstd[(int64_t)row * g.groups + blockIdx.y] = r;
    A* y = static_cast<A*>(g.y) + (int64_t)row * g.width + c0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float o[8], rr[8], wf[8];
      w[c].floats(wf);
      vset(rr, r);
      vmul(o, h[c], rr);
      vmul(o, o, wf);
      Eight<A> to;
      to.set(o);
      store_chunk<LAY>(to, y, c, left);
    }
  }
  if constexpr (kRing) asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace

void check_norm(const fhe_rms_norm_args& a) {
  require(a.dtype == FHE_F32 || a.dtype == FHE_BF16 || a.dtype == FHE_F16, "dtype must be FHE_F32, FHE_BF16 or FHE_F16");
  require(!a.gate || !a.residual, "a norm has a residual or a gate, not both");
  require(a.gate || a.stream_dtype == a.dtype || a.stream_dtype == FHE_F32, "stream_dtype must be dtype or FHE_F32");
  require(a.groups >= 1 && a.width >= 1 && a.width % a.groups == 0, "width must be a positive multiple of groups");
  require(a.gate || a.groups == 1, "groups need a gate");
  require(a.width / a.groups <= kMaxNormWidth, "a group must have at most 16384 channels");
  require(a.groups <= 65535 && a.width < (1u << 30) && a.rows < (1u << 31) &&
              (uint64_t)a.rows * a.groups < (1ull << 31),
          "sizes too large");
  require(a.eps > 0.f && a.eps < INFINITY, "eps must be positive");
  require(!a.channel_scale || a.residual, "channel_scale needs a residual");
  require(a.scale - a.scale == 0.f, "scale must be finite");
}

NormArgs norm_args(const fhe_rms_norm_args& a) {
  NormArgs g{};
  g.x = a.x;
  g.xs = a.x_stride;
  g.res = a.residual;
  g.rs = a.residual_stride;
  g.gate = a.gate;
  g.gs = a.gate_stride;
  g.cscale = a.channel_scale;
  g.weight = a.weight;
  g.y = a.y;
  g.h = a.h;
  g.rstd = a.rstd;
  g.rows = a.rows;
  g.width = a.width;
  g.groups = a.groups;
  g.gw = a.width / a.groups;
  g.eps = a.eps;
  g.scale = a.scale;
  return g;
}

void rms_norm(const fhe_rms_norm_args& a) {
  check_norm(a);
  if (a.rows == 0) return;
  require(a.x && a.weight && a.y && (!a.residual || a.h), "null input or output");
  DeviceGuard dev(a.device);
  NormArgs g = norm_args(a);
  const uint32_t ea = elem_size(a.dtype), eh = a.gate ? ea : elem_size(a.stream_dtype);
  const uint32_t ex = a.gate || a.residual ? ea : eh;
  Together t(g.gw);
  t.with(a.x, a.x_stride, ex);
  if (a.residual) t.with(a.residual, a.residual_stride, eh);
  if (a.gate) t.with(a.gate, a.gate_stride, ea);
  t.with(a.channel_scale, 0, 4);
  t.with(a.weight, 0, 4);
  t.with(a.y, a.width, ea);
  t.with(a.h, a.width, eh);
  const NormShape s = norm_shape(g.gw, (uint64_t)a.rows * a.groups, t.n);
  g.lanes = s.lanes;
  // blocks that go from row to row
  uint32_t resident = 12, shared = 0;
  if (a.gate && s.layout(t.n) == kWords) {
    const uint32_t warps = s.warps * s.rows_per_block, row = s.chunks * ea * 16 * 32 * warps;
    const RingPlan r = ring_plan(row, warps, 104 * 1024);
    g.stages = (int)r.stages;
    shared = r.stages * row;
    resident = r.blocks;
  }
  const uint32_t blocks = std::min((a.rows + s.rows_per_block - 1) / s.rows_per_block,
                                   std::max(1u, 148 * resident / a.groups));
  with_norm(a, s.chunks, s.layout(t.n), [&](auto mode, auto act, auto str, auto chunks, auto layout) {
    auto k = k_norm<decltype(mode)::value, decltype(act), decltype(str), decltype(chunks)::value, decltype(layout)::value>;
    if (shared > 48000) allow_shared(k, kSmShared - kBlockShared);
    const dim3 block(32 * s.warps, s.warps == 1 ? 4 : 1);
    k<<<dim3(blocks, a.groups), block, shared, static_cast<cudaStream_t>(a.stream)>>>(g);
  });
  note_launch();
  FHE_CUDA(cudaGetLastError());
}

}  // namespace fhe
