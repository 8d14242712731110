// Root-mean-square norms with their residual or their gate (fhe_rms_norm).
//
// y = h r w with r = 1 / sqrt(mean(h^2) + eps) over a row, or over each group of a
// row, of h = x, residual + scale x (stored in the stream's type, which is what
// the norm is of) or x SiLU(gate).  A row lies in the registers of one to sixteen
// warps, eight channels to a 16-byte word, so its inputs are read once and its
// outputs written once: memory bounds it.  The weights stay in registers while a
// block goes from row to row.
#include "launch_count.h"
#include "norms.h"

namespace fhe {
namespace {

template <int MODE, class A, class H, int N, bool VEC>
__global__ void __launch_bounds__(512) k_norm(const NormArgs g) {
  __shared__ float red[2][16];
  RowSum row_sum{red};
  using X = std::conditional_t<MODE == kNormPlain, H, A>;
  const uint32_t gw = g.gw, c0 = blockIdx.y * gw;
  float w[N][8];
  float cs[MODE == kNormAddScaled ? N : 1][8];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    Eight<float> e;
    load_chunk<VEC>(e, g.weight + c0, c, gw);
    e.floats(w[c]);
    if constexpr (MODE == kNormAddScaled) {
      load_chunk<VEC>(e, g.cscale + c0, c, gw);
      e.floats(cs[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) cs[c][i] *= g.scale;
    }
  }
  const float n = 1.f / (float)gw;
  // the next row's words come while this one is summed and written
  constexpr bool kTwo = MODE != kNormPlain;
  using Y = std::conditional_t<MODE == kNormGate, A, H>;  // gate or residual
  Eight<X> e[N];
  Eight<Y> f[kTwo ? N : 1];
  auto fetch = [&](uint32_t row) {
    const X* x = static_cast<const X*>(g.x) + (int64_t)row * g.xs + c0;
    const Y* y = MODE == kNormGate ? static_cast<const Y*>(g.gate) + (int64_t)row * g.gs + c0
                                   : static_cast<const Y*>(g.res) + (int64_t)row * g.rs + c0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      load_chunk<VEC>(e[c], x, c, gw);
      if constexpr (kTwo) load_chunk<VEC>(f[c], y, c, gw);
    }
  };
  const uint32_t step = gridDim.x * blockDim.y;
  uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
  if (row < g.rows) fetch(row);
  for (; row < g.rows; row += step) {
    float h[N][8];
    [[maybe_unused]] H* out = static_cast<H*>(g.h) + (int64_t)row * g.width + c0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if constexpr (MODE == kNormPlain) {
        e[c].floats(h[c]);
      } else if constexpr (MODE == kNormGate) {
        float q[8], zf[8];
        f[c].floats(zf);
        sigmoid(q, zf);
        e[c].floats(h[c]);
        vmul(q, q, zf);
        vmul(h[c], h[c], q);
      } else {
        float xf[8], rf[8], s[8];
        e[c].floats(xf);
        f[c].floats(rf);
        if constexpr (MODE == kNormAddScaled) vfma(h[c], cs[c], xf, rf);
        else vset(s, g.scale), vfma(h[c], s, xf, rf);
        Eight<H> kept;
        kept.set(h[c]);
        store_chunk<VEC>(kept, out, c, gw);
        kept.floats(h[c]);
      }
    }
    if (row + step < g.rows) fetch(row + step);
    float part[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float p[2] = {h[c][i], h[c][i + 1]};
        vfma(part, p, p, part);
      }
    const float ss = row_sum(part[0] + part[1]);
    float r = 1.f / sqrtf(fmaf(ss, n, g.eps));
    // squares past fp32's range: the row again, scaled (an infinity of the row itself gives r = 0)
    if (ss == INFINITY) {
      const float k = 0x1p-80f;
      float again = 0.f;
#pragma unroll
      for (int c = 0; c < N; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) again = fmaf(h[c][i] * k, h[c][i] * k, again);
      r = k / sqrtf(row_sum(again) * n);
    }
    if (g.rstd && threadIdx.x == 0) g.rstd[(int64_t)row * g.groups + blockIdx.y] = r;
    A* y = static_cast<A*>(g.y) + (int64_t)row * g.width + c0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float o[8], rr[8];
      vset(rr, r);
      vmul(o, h[c], rr);
      vmul(o, o, w[c]);
      Eight<A> e;
      e.set(o);
      store_chunk<VEC>(e, y, c, gw);
    }
  }
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
  const NormArgs g = norm_args(a);
  const uint32_t ea = elem_size(a.dtype), eh = a.gate ? ea : elem_size(a.stream_dtype);
  const uint32_t ex = a.gate || a.residual ? ea : eh;
  const bool vec = g.gw % 8 == 0 && norm_aligned(a.x, a.x_stride, ex) && norm_aligned(a.residual, a.residual_stride, eh) &&
                   norm_aligned(a.gate, a.gate_stride, ea) && norm_aligned(a.channel_scale, 0, 4) &&
                   norm_aligned(a.weight, 0, 4) && norm_aligned(a.y, 0, ea) && norm_aligned(a.h, 0, eh);
  const NormShape s = norm_shape(g.gw, (uint64_t)a.rows * a.groups, vec);
  const uint32_t blocks = std::min((a.rows + s.rows_per_block - 1) / s.rows_per_block,
                                   std::max(1u, 148 * 12 / a.groups));
  with_norm(a, s.chunks, vec, [&](auto mode, auto act, auto str, auto chunks, auto words) {
    k_norm<decltype(mode)::value, decltype(act), decltype(str), decltype(chunks)::value, decltype(words)::value>
        <<<dim3(blocks, a.groups), dim3(32 * s.warps, s.rows_per_block), 0, static_cast<cudaStream_t>(a.stream)>>>(g);
  });
  note_launch();
  FHE_CUDA(cudaGetLastError());
}

}  // namespace fhe
