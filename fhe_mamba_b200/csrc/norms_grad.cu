// Gradients of the root-mean-square norms (fhe_rms_norm_backward).
//
// With a = dy w and u = h r: dh = r (a - u mean(a u)) (+ the gradient that h
// itself has), dweight = sum over rows of dy u.  Like the norm, a row is spread
// over one to sixteen warps and read once.  Its words come by asynchronous copies
// through each thread's own part of shared memory, rows ahead, and are taken from
// there twice, for the mean and for the gradients; single elements are held in
// registers.  A block keeps its share of the sums over rows in registers from row
// to row, and a second launch adds the blocks' shares in a fixed order.
#include "launch_count.h"
#include "norms.h"

namespace fhe {
namespace {

// Through the first cache where a thread's two words of float32 lie in one sector,
// past it otherwise.
template <bool TWO>
__device__ __forceinline__ void copy16(void* to, const void* from) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (TWO) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
}

// A thread's share of a row in shared memory, in 16-byte words: what is read twice
// stays out of the registers, and the loads of the next rows run behind the
// arithmetic of this one.
template <int MODE, class A, class H, int N>
struct GradRing {
  static constexpr bool kAdd = MODE == kNormAdd || MODE == kNormAddScaled;
  static constexpr int kWa = sizeof(A) / 2, kWs = (MODE == kNormGate ? sizeof(A) : sizeof(H)) / 2, kWh = sizeof(H) / 2;
  static constexpr int kS = 0, kDy = kS + N * kWs, kZ = kDy + N * kWa,
                       kDh = kZ + (MODE == kNormGate || MODE == kNormAddScaled ? N * kWa : 0),
                       kWords = kDh + (kAdd ? N * kWh : 0);
};

template <int MODE, class A, class H, int N, bool VEC>
__global__ void __launch_bounds__(N == 3 ? 256 : 512) k_norm_grad(const NormArgs g) {
  __shared__ float red[2][16];
  extern __shared__ __align__(16) float sums[];  // the ring of rows; then sums over a block's rows
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
  // what a row is read from: h or x, dy, gate or (for the channel scale) x, dh
  constexpr bool kThird = MODE == kNormGate || kScaled;
  using Ring = GradRing<MODE, A, H, N>;
  Eight<S> s[VEC ? 1 : N];
  Eight<A> dy[VEC ? 1 : N], z[kThird && !VEC ? N : 1];
  Eight<H> dh[kAdd && !VEC ? N : 1];
  uint8_t* ring = reinterpret_cast<uint8_t*>(sums) + (threadIdx.y * blockDim.x + threadIdx.x) * 16;
  auto visit = [&](uint32_t row, int stage, auto&& f_s, auto&& f_dy, auto&& f_z, auto&& f_dh) {
    const int64_t out = (int64_t)row * g.width + c0;
    const S* src = kAdd ? static_cast<const S*>(g.h) + out : static_cast<const S*>(g.x) + (int64_t)row * g.xs + c0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      f_s(src, c);
      f_dy(static_cast<const A*>(g.dy) + out, c);
      if constexpr (MODE == kNormGate) f_z(static_cast<const A*>(g.gate) + (int64_t)row * g.gs + c0, c);
      if constexpr (kScaled) f_z(static_cast<const A*>(g.x) + (int64_t)row * g.xs + c0, c);
      if constexpr (kAdd)
        if (g.dh) f_dh(static_cast<const H*>(g.dh) + out, c);
    }
  };
  const uint32_t step = gridDim.x * blockDim.y, row0 = blockIdx.x * blockDim.y + threadIdx.y;
  const uint32_t threads = blockDim.x * blockDim.y;
  auto fetch = [&](uint32_t row, int stage) {
    if constexpr (VEC) {
      if (row < g.rows) {
        auto copy = [&](int first) {
          return [&, first](const auto* p, int c) {
            constexpr int W = sizeof(*p) / 2;  // 16-byte words of a chunk
            const uint32_t at = channel<true>(c, 0);
#pragma unroll
            for (int k = 0; k < W; ++k)
              if (at < gw) copy16<W == 2>(ring + (uint64_t)(stage * Ring::kWords + first + c * W + k) * threads * 16, p + at + k * (8 / W));
          };
        };
        visit(row, stage, copy(Ring::kS), copy(Ring::kDy), copy(Ring::kZ), copy(Ring::kDh));
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    } else if (row < g.rows) {
      visit(row, 0, [&](const S* p, int c) { load_chunk<VEC>(s[c], p, c, gw); },
            [&](const A* p, int c) { load_chunk<VEC>(dy[c], p, c, gw); },
            [&](const A* p, int c) { load_chunk<VEC>(z[c], p, c, gw); },
            [&](const H* p, int c) { load_chunk<VEC>(dh[c], p, c, gw); });
    }
  };
  const int stages = g.stages;
  int stage = 0;
  // chunk c of an array, from the ring or the registers; lanes past the row hold 0
  auto take = [&](auto* held, int first, int c, float (&o)[8]) {
    using T = std::remove_pointer_t<decltype(held)>;
    if constexpr (VEC) {
      constexpr int W = sizeof(T) / 16;
      T e;
#pragma unroll
      for (int k = 0; k < W; ++k)
        reinterpret_cast<uint4*>(&e)[k] = channel<true>(c, 0) < gw
            ? *reinterpret_cast<const uint4*>(ring + (uint64_t)(stage * Ring::kWords + first + c * W + k) * threads * 16)
            : make_uint4(0, 0, 0, 0);
      e.floats(o);
    } else {
      held[c].floats(o);
    }
  };
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (i + 1 < stages) fetch(row0 + i * step, i);
  }
  for (uint32_t row = row0; row < g.rows; row += step) {
    const int64_t out = (int64_t)row * g.width + c0;
    if constexpr (VEC) {
      fetch(row + (stages - 1) * step, stage ? stage - 1 : stages - 1);
      if (stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
      else if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
      fetch(row, 0);
    }
    const float r = g.rstd[(int64_t)row * g.groups + blockIdx.y];
    float rr[8];
    vset(rr, r);
    // u = h r; with a gate also p = SiLU(gate)
    auto unit = [&](int c, float (&u)[8], float (&xf)[8], float (&p)[8], float (&q)[8], float (&zf)[8]) {
      take(s, Ring::kS, c, xf);
      if constexpr (MODE == kNormGate) {
        take(z, Ring::kZ, c, zf);
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
      take(dy, Ring::kDy, c, d);
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
      take(dy, Ring::kDy, c, d);
      vmul(d, d, w[c]);
      vfma(d, u, mm, d);
      if constexpr (kAdd) {
        float e[8];
        vset(e, 0.f);
        if (g.dh) take(dh, Ring::kDh, c, e);
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
          take(z, Ring::kZ, c, xg);
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
    stage = stage + 1 == stages ? 0 : stage + 1;
  }
  if constexpr (VEC) asm volatile("cp.async.wait_all;" ::: "memory");
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

// How a call is laid out: shape, rows of the ring (up to three, as far as 12 warps
// still fit an SM), shared memory, and blocks that go from row to row, as many as
// are resident.
struct GradPlan {
  NormShape shape;
  bool vec;
  uint32_t stages, shared, blocks;
};
GradPlan grad_plan(const fhe_rms_norm_grad_args& a) {
  constexpr uint32_t kShared = 227 * 1024, kOwn = 1024 + 128;  // of an SM; of a block beside its ring
  const fhe_rms_norm_args& f = a.f;
  const uint32_t gw = f.width / f.groups;
  const uint32_t wa = elem_size(f.dtype) / 2, wh = f.gate ? wa : elem_size(f.stream_dtype) / 2;
  const uint32_t per_chunk = (f.gate ? wa : wh) + wa + (f.gate || f.channel_scale ? wa : 0) + (f.residual ? wh : 0);
  GradPlan p{};
  p.vec = words(a);
  for (;; p.vec = false) {
    p.shape = norm_shape(gw, (uint64_t)f.rows * f.groups, p.vec);
    const uint32_t warps = p.shape.warps * p.shape.rows_per_block;
    uint32_t resident = std::max(1u, 16 / warps);
    p.shared = p.shape.rows_per_block > 1 ? gw * sizeof(float) : 0;  // one warp's channels, at most 1024
    if (p.vec) {
      const uint32_t row = p.shape.chunks * per_chunk * 16 * 32 * warps;
      if (row + kOwn > kShared) continue;
      for (p.stages = 3; p.stages > 1; --p.stages) {
        const uint32_t fit = kShared / (p.stages * row + kOwn);
        if (fit && fit * warps >= 12) break;
      }
      p.shared = std::max(p.shared, p.stages * row);
      resident = std::max(1u, std::min(resident, kShared / (p.shared + kOwn)));
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
  return (uint64_t)grad_plan(a).blocks * a.f.width * sizeof(float) * (a.f.channel_scale ? 2 : 1);
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
  const GradPlan p = grad_plan(a);
  g.stages = (int)p.stages;
  with_norm(f, p.shape.chunks, p.vec, [&](auto mode, auto act, auto str, auto chunks, auto words) {
    auto k = k_norm_grad<decltype(mode)::value, decltype(act), decltype(str), decltype(chunks)::value,
                         decltype(words)::value>;
    if (p.shared > 48000) FHE_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.shared));
    k<<<dim3(p.blocks, f.groups), dim3(32 * p.shape.warps, p.shape.rows_per_block), p.shared, st>>>(g);
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
