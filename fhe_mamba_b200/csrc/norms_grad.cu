// Gradients of the root-mean-square norms (fhe_rms_norm_backward).
//
// With a = dy w and u = h r: dh = r (a - u mean(a u)) (+ the gradient that h
// itself has), dweight = sum over rows of dy u.  Like the norm, a row lies in
// registers and is read once; a block keeps its share of the sums over rows in
// registers from row to row, and a second launch adds the blocks' shares in a
// fixed order.
#include "launch_count.h"
#include "norms.h"

namespace fhe {
namespace {

template <int MODE, class A, class H, int N, bool VEC>
__global__ void __launch_bounds__(N == 3 ? 256 : 512) k_norm_grad(const NormArgs g) {
  __shared__ float red[2][16];
  extern __shared__ float sums[];  // [channels of the group]
  RowSum row_sum{red};
  constexpr bool kAdd = MODE == kNormAdd || MODE == kNormAddScaled, kScaled = MODE == kNormAddScaled;
  using X = std::conditional_t<MODE == kNormPlain, H, A>;  // x
  using S = std::conditional_t<MODE == kNormGate, A, H>;   // what h is made from
  const uint32_t gw = g.gw, c0 = blockIdx.y * gw;
  float w[N][8], dw[N][8];
  float cs[kScaled ? N : 1][8], dcs[kScaled ? N : 1][8];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    Eight<float> e;
    load_chunk<VEC>(e, g.weight + c0, c, gw);
    e.floats(w[c]);
    vset(dw[c], 0.f);
    if constexpr (kScaled) {
      load_chunk<VEC>(e, g.cscale + c0, c, gw);
      e.floats(cs[c]);
      vset(dcs[c], 0.f);
    }
  }
  const float n = 1.f / (float)gw;
  for (uint32_t row = blockIdx.x * blockDim.y + threadIdx.y; row < g.rows; row += gridDim.x * blockDim.y) {
    const int64_t out = (int64_t)row * g.width + c0;
    const S* src = kAdd ? static_cast<const S*>(g.h) + out : static_cast<const S*>(g.x) + (int64_t)row * g.xs + c0;
    const A* dyp = static_cast<const A*>(g.dy) + out;
    Eight<S> s[N];
    Eight<A> dy[N], z[MODE == kNormGate || kScaled ? N : 1];
    Eight<H> dh[kAdd ? N : 1];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      load_chunk<VEC>(s[c], src, c, gw);
      load_chunk<VEC>(dy[c], dyp, c, gw);
      if constexpr (MODE == kNormGate) load_chunk<VEC>(z[c], static_cast<const A*>(g.gate) + (int64_t)row * g.gs + c0, c, gw);
      if constexpr (kScaled) load_chunk<VEC>(z[c], static_cast<const A*>(g.x) + (int64_t)row * g.xs + c0, c, gw);
      if constexpr (kAdd)
        if (g.dh) load_chunk<VEC>(dh[c], static_cast<const H*>(g.dh) + out, c, gw);
    }
    const float r = g.rstd[(int64_t)row * g.groups + blockIdx.y];
    float rr[8];
    vset(rr, r);
    // u = h r; with a gate also p = SiLU(gate)
    auto unit = [&](int c, float (&u)[8], float (&xf)[8], float (&p)[8], float (&q)[8], float (&zf)[8]) {
      s[c].floats(xf);
      if constexpr (MODE == kNormGate) {
        z[c].floats(zf);
        sigmoid(q, zf);
        vmul(p, q, zf);
        vmul(u, xf, p);
        vmul(u, u, rr);
      } else {
        vmul(u, xf, rr);
      }
    };
    float part[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float u[8], xf[8], p[8], q[8], zf[8], d[8], a[8];
      unit(c, u, xf, p, q, zf);
      dy[c].floats(d);
      vmul(a, d, u);
      vadd(dw[c], dw[c], a);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float aa[2] = {a[i], a[i + 1]}, ww[2] = {w[c][i], w[c][i + 1]};
        vfma(part, aa, ww, part);
      }
    }
    const float m = row_sum(part[0] + part[1]) * n;
    float mm[8];
    vset(mm, -m);
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float u[8], xf[8], p[8], q[8], zf[8], d[8];
      unit(c, u, xf, p, q, zf);
      dy[c].floats(d);
      vmul(d, d, w[c]);
      vfma(d, u, mm, d);
      if constexpr (kAdd) {
        float e[8];
        vset(e, 0.f);
        if (g.dh) dh[c].floats(e);
        vfma(d, d, rr, e);
      } else {
        vmul(d, d, rr);
      }
      if constexpr (MODE == kNormGate) {
        float o[8], one[8];
        Eight<A> e;
        vmul(o, d, p);
        e.set(o);
        if (g.dx) store_chunk<VEC>(e, static_cast<A*>(g.dx) + out, c, gw);
        // SiLU' = q (1 + z (1 - q)) = q + p (1 - q)
#pragma unroll
        for (int i = 0; i < 8; ++i) one[i] = 1.f - q[i];
        vfma(o, p, one, q);
        vmul(d, d, xf);
        vmul(o, o, d);
        e.set(o);
        if (g.dgate) store_chunk<VEC>(e, static_cast<A*>(g.dgate) + out, c, gw);
      } else {
        if constexpr (kScaled) {
          float xg[8];
          z[c].floats(xg);
          vfma(dcs[c], d, xg, dcs[c]);
        }
        if constexpr (kAdd) {
          Eight<H> e;
          e.set(d);
          if (g.dres) store_chunk<VEC>(e, static_cast<H*>(g.dres) + out, c, gw);
          float sc[8];
          vset(sc, g.scale);
          vmul(d, d, sc);
          if constexpr (kScaled) vmul(d, d, cs[c]);
        }
        Eight<X> e;
        e.set(d);
        if (g.dx) store_chunk<VEC>(e, static_cast<X*>(g.dx) + out, c, gw);
      }
    }
  }
  // the block's rows together, one after the other
  auto gather = [&](float (&v)[N][8], float* to, float k) {
    for (uint32_t turn = 0; turn < blockDim.y; ++turn) {
      __syncthreads();
      if (threadIdx.y != turn) continue;
#pragma unroll
      for (int c = 0; c < N; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t at = channel<VEC>(c, i);
          if (at >= gw) continue;
          const float sum = turn ? sums[at] + v[c][i] : v[c][i];
          if (turn + 1 == blockDim.y) to[at] = sum * k;
          else sums[at] = sum;
        }
    }
  };
  if (g.part) {
    float* to = g.part + (int64_t)blockIdx.x * g.width + c0;
    gather(dw, to, 1.f);
    if constexpr (kScaled) gather(dcs, to + (int64_t)gridDim.x * g.width, g.scale);
  }
}

// Adds the blocks' shares: 32 channels x 16 strands of blocks.
__global__ void __launch_bounds__(512) k_norm_sum(const float* part, uint32_t blocks, uint32_t width, float* dweight,
                                                  float* dcscale) {
  __shared__ float s[16][33];
  const uint32_t c = blockIdx.x * 32 + threadIdx.x;
  float* out = blockIdx.y ? dcscale : dweight;
  if (!out) return;
  part += (int64_t)blockIdx.y * blocks * width;
  float v = 0.f;
  if (c < width) {
#pragma unroll 8
    for (uint32_t b = threadIdx.y; b < blocks; b += 16) v += part[(int64_t)b * width + c];
  }
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    for (int i = 1; i < 16; ++i) v += s[i][threadIdx.x];
    out[c] = v;
  }
}

bool words(const fhe_rms_norm_grad_args& a) {
  const fhe_rms_norm_args& f = a.f;
  const uint32_t ea = elem_size(f.dtype), eh = f.gate ? ea : elem_size(f.stream_dtype);
  const uint32_t ex = f.gate || f.residual ? ea : eh;
  const bool x_read = !f.residual || f.channel_scale;
  return f.width / f.groups % 8 == 0 && (!x_read || norm_aligned(f.x, f.x_stride, ex)) &&
         (!f.residual || norm_aligned(f.h, 0, eh)) && norm_aligned(f.gate, f.gate_stride, ea) &&
         norm_aligned(f.channel_scale, 0, 4) && norm_aligned(f.weight, 0, 4) && norm_aligned(a.dy, 0, ea) &&
         norm_aligned(a.dh, 0, eh) && norm_aligned(a.dx, 0, ex) && norm_aligned(a.dresidual, 0, eh) &&
         norm_aligned(a.dgate, 0, ea);
}

NormShape grad_shape(const fhe_rms_norm_grad_args& a) {
  return norm_shape(a.f.width / a.f.groups, (uint64_t)a.f.rows * a.f.groups, words(a), true);
}

// Blocks that go from row to row: 16 warps an SM.
uint32_t grad_blocks(const fhe_rms_norm_grad_args& a, const NormShape& s) {
  const uint32_t resident = std::max(1u, 16 / (s.warps * s.rows_per_block));
  return std::max(1u, std::min((a.f.rows + s.rows_per_block - 1) / s.rows_per_block,
                               std::max(1u, 148 * resident / a.f.groups)));
}

bool sums_wanted(const fhe_rms_norm_grad_args& a) { return a.dweight || a.dchannel_scale; }

}  // namespace

uint64_t rms_norm_backward_workspace(const fhe_rms_norm_grad_args& a) {
  check_norm(a.f);
  if (!sums_wanted(a)) return 0;
  return (uint64_t)grad_blocks(a, grad_shape(a)) * a.f.width * sizeof(float) * (a.f.channel_scale ? 2 : 1);
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
  const bool vec = words(a);
  const NormShape s = grad_shape(a);
  const uint32_t blocks = grad_blocks(a, s);
  const size_t shared = s.rows_per_block > 1 ? g.gw * sizeof(float) : 0;  // at most 1024 channels: one warp's
  with_norm(f, s.chunks, vec, [&](auto mode, auto act, auto str, auto chunks, auto words) {
    k_norm_grad<decltype(mode)::value, decltype(act), decltype(str), decltype(chunks)::value, decltype(words)::value>
        <<<dim3(blocks, f.groups), dim3(32 * s.warps, s.rows_per_block), shared, st>>>(g);
  });
  note_launch();
  if (g.part) {
    k_norm_sum<<<dim3((f.width + 31) / 32, f.channel_scale ? 2 : 1), dim3(32, 16), 0, st>>>(
        g.part, blocks, f.width, a.dweight, a.dchannel_scale);
    note_launch();
  }
  FHE_CUDA(cudaGetLastError());
}

}  // namespace fhe
