// Mamba-2 state recurrence for bfloat16 activations on the tensor cores
// (tcgen05.mma kind::f16), 128 tokens at a time.
//
// The walk of mamba_scan.cu, o_t = S_t q_t with S_t = a_t S_(t-1) + w_t r_t (x) k_t,
// over a chunk of 128 tokens from a carried state S0 is four products:
//   G  = q k^T                                     [t][s], 128 x 128 over the columns
//   O  = (G o L o w) r  +  P_t (q S0^T)            [t][r], L_ts = prod of a over (s, t], P_t over [0, t]
//   S' = P_end S0 + k^T (E o w o r)                [c][r], E_t = prod of a over (t, end]
// and reversed in time (dS_t = a_(t+1) dS_(t+1) + r_t (x) k_t) the same with
// L_ts = prod over (t, s], P_t over (t, end], E_t over [0, t].
// Every factor is a product of at most 128 decays in its own order, never a
// quotient, so decays of zero or near it lose nothing.
//
// Roundings.  q, k and r are bfloat16 as given; G, O and S accumulate in
// fp32.  G o L o w and S0 enter their products as bfloat16, half a step of
// 2^-8 of each term, as y's own rounding; with PRECISE they enter as two
// bfloat16 terms (2^-16).  E o w o r, whose sum is the fp32 state, always
// enters as two terms.
//
// One CTA walks one (batch, head, 64 rows, segment).  Shared memory holds q,
// k, r and S0 in 128-byte-swizzled tiles of 64 columns; the scaled r takes
// q's place once q has been used, which keeps two CTAs on an SM, so that one
// computes while the other waits for its loads or its products.  Tensor
// memory: G (its columns become the A operand G o L o w), O and S'.  The state
// itself stays in registers.
#include <algorithm>

#include "launch_count.h"
#include "mamba_ops.h"
#include "mamba_scan.h"

namespace fhe {
namespace {

constexpr uint32_t kQ = 128;            // tokens per chunk (MMA M)
constexpr uint32_t kRowsTc = 64;        // rows per CTA (MMA N)
constexpr uint32_t kThreadsTc = 256;
constexpr uint32_t kTile = kQ * 128;    // bytes of a 128 x 64 tile
constexpr uint32_t kTmemCols = 256;     // G 128, O 64, S' 64
constexpr uint32_t kColO = 128, kColS = 192;
// More than a third of an SM's shared memory: at most two CTAs are resident,
// whose tensor memory (2 x 256 columns) fits.
constexpr uint32_t kLeastSmem = 80 * 1024;
// Bound on a wait for an MMA group, far above its microseconds; on expiry the
// kernel counts the failure, leaves its outputs and frees its tensor memory.
constexpr uint32_t kWaitLimit = 1u << 20;

__device__ unsigned g_scan_timeouts = 0;

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 128-byte-swizzled tiles: 8-row groups 1024 bytes apart; for operands whose
// M or N axis is the contiguous one, the next 64 of it `lead` bytes on.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lead >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kind::f16, bfloat16 operands, fp32 accumulator; a_mn / b_mn: the operand's
// M / N axis is contiguous.
constexpr uint32_t idesc(uint32_t n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) |
         ((kQ >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc));
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 columns of this warp's 32 lanes; the caller waits (ld_wait) before using them.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
__device__ __forceinline__ void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 bytes to shared memory, the first `bytes` of them from src and zeros after.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t v;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}
__device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
// The two bfloat16 terms of a pair of floats.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2(a, b);
  lo = pack2(a - low(hi), b - high(hi));
}

// Byte offset of 16-byte word `word` of row `row` in a 128-byte-swizzled tile.
__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t word) { return row * 128 + ((word ^ (row & 7)) << 4); }

struct Gates {
  float a[kQ], w[kQ];    // decay and write of each token
  float head[kQ];        // product over its block of 32 up to and with the token
  float tail[kQ];        // product over its block after the token
  float col[kQ];         // the column factor times w: tail (forward) or head (reversed)
  float total[4];        // product over each block
};

// One block of 32 columns of G o L o w for one row, in place in v; `own` is
// the row's own block.  `scale` multiplies the row (it is in `row` already).
template <bool REV>
__device__ __forceinline__ void weigh(float (&v)[32], const Gates& g, uint32_t blk, bool own, uint32_t lane, float row,
                                      float scale) {
  const uint32_t s0 = blk * 32;
  if (!own) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 c = *reinterpret_cast<const float4*>(&g.col[s0 + i]);
      v[i] *= row * c.x;
      v[i + 1] *= row * c.y;
      v[i + 2] *= row * c.z;
      v[i + 3] *= row * c.w;
    }
    return;
  }
  float p = 1.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    if constexpr (!REV) {
      const int i = 31 - j;  // p = product of a over (i, lane]
      if (i < 31) p = i < (int)lane ? p * g.a[s0 + i + 1] : 1.f;
      v[i] = i <= (int)lane ? v[i] * (scale * (p * g.w[s0 + i])) : 0.f;
    } else {
      const int i = j;       // p = product of a over (lane, i]
      p = i > (int)lane ? p * g.a[s0 + i] : 1.f;
      v[i] = i >= (int)lane ? v[i] * (scale * (p * g.w[s0 + i])) : 0.f;
    }
  }
}

// COLS: columns held, 64 or 128 (those past g.cols are zeros).
template <int COLS, bool REV, int OUT, bool PRECISE>
__global__ void __launch_bounds__(kThreadsTc, 2) k_scan_tc(const RecArgs g) {
  constexpr uint32_t kHalves = COLS / 64;
  constexpr uint32_t kBytesK = kHalves * kTile;
  constexpr uint32_t kBytesS = COLS * 128;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Gates gate;
  __shared__ __align__(8) uint64_t bars[3];  // G and q S0, S', O
  __shared__ uint32_t tslot;
  const uint32_t sq = smem_u32(smem);            // q, then the scaled r (two terms)
  const uint32_t sk = sq + 2 * kTile;
  const uint32_t sr = sk + kBytesK;
  const uint32_t ss = sr + kTile;                // S0 (two terms with PRECISE)
  const uint32_t bar_g = smem_u32(&bars[0]), bar_s = bar_g + 8, bar_o = bar_g + 16;

  const uint32_t tiles = (g.rows + kRowsTc - 1) / kRowsTc;
  uint32_t id = blockIdx.x;
  const uint32_t row0 = id % tiles * kRowsTc;
  id /= tiles;
  const uint32_t h = id % g.heads;
  id /= g.heads;
  const uint32_t seg = id % g.nseg, b = id / g.nseg;
  const int64_t bh = (int64_t)b * g.heads + h;
  const int len = clamp_length(g.lengths, b, g.length);
  const int t_lo = seg * g.seglen, t_hi = min(t_lo + (int)g.seglen, (int)g.length);
  const int chunks = (t_hi - t_lo + (int)kQ - 1) / (int)kQ;

  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t quarter = warp & 3, half = warp >> 2;
  const uint32_t t = quarter * 32 + lane;  // this thread's token, and column of S
  using T = __nv_bfloat16;
  const T* rp = g.r.at<T>(b, h) + row0;
  const T* kp = g.k.at<T>(b, h);
  const T* qp = g.q.at<T>(b, h);

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tslot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 0) {
    for (int i = 0; i < 3; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar_g + 8 * i));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }

  auto first = [&](int i) { return REV ? t_hi - (int)kQ * (i + 1) : t_lo + (int)kQ * i; };
  auto live = [&](int tok) { return tok >= t_lo && tok < t_hi && tok < len; };
  // A [128][COLS] tile: 16-byte words, columns past `cols` and dead tokens zero.
  auto load_cols = [&](uint32_t dst, const T* p, int64_t sl, int t0) {
#pragma unroll
    for (uint32_t e = tid; e < kQ * COLS / 8; e += kThreadsTc) {
      const uint32_t row = e / (COLS / 8), word = e % (COLS / 8);
      const int tok = t0 + (int)row, col = (int)word * 8;
      const int n = live(tok) ? min(max(((int)g.cols - col) * 2, 0), 16) : 0;
      copy16(dst + (word >> 3) * kTile + swz(row, word & 7), n ? p + (int64_t)tok * sl + col : p, n);
    }
  };
  auto load_rows = [&](int t0) {
#pragma unroll
    for (uint32_t e = tid; e < kQ * 8; e += kThreadsTc) {
      const uint32_t row = e / 8, word = e % 8;
      const int tok = t0 + (int)row, col = (int)word * 8;
      const int n = live(tok) ? min(max(((int)g.rows - (int)row0 - col) * 2, 0), 16) : 0;
      copy16(sr + swz(row, word), n ? rp + (int64_t)tok * g.r.sl + col : rp, n);
    }
  };
  auto load_kq = [&](int t0) {
    load_cols(sk, kp, g.k.sl, t0);
    if constexpr (OUT != kOutNone) load_cols(sq, qp, g.q.sl, t0);
  };

  // The state: column t of rows half * 32 + i.
  float s[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t row = row0 + half * 32 + i;
    s[i] = (OUT != kOutNone && g.state_in && row < g.rows && t < g.cols)
               ? g.state_in[bh * g.in_bh + seg * g.in_seg + row * g.st_row + t * g.st_col]
               : 0.f;
  }
  auto put_state = [&] {  // S0 as the B operand [column][row]
    if (t >= (uint32_t)COLS) return;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      uint4 hi, lo;
      split2(s[8 * v], s[8 * v + 1], hi.x, lo.x);
      split2(s[8 * v + 2], s[8 * v + 3], hi.y, lo.y);
      split2(s[8 * v + 4], s[8 * v + 5], hi.z, lo.z);
      split2(s[8 * v + 6], s[8 * v + 7], hi.w, lo.w);
      const uint32_t at = ss - sq + swz(t, half * 4 + v);
      *reinterpret_cast<uint4*>(smem + at) = hi;
      if constexpr (PRECISE) *reinterpret_cast<uint4*>(smem + at + kBytesS) = lo;
    }
  };
  if constexpr (OUT != kOutNone) put_state();
  load_kq(first(0));
  load_rows(first(0));

  const float* wp = g.write.p ? g.write.p + (int64_t)b * g.write.sb + (int64_t)h * g.write.sh : nullptr;
  const float* ap = g.log_decay.p + (int64_t)b * g.log_decay.sb + (int64_t)h * g.log_decay.sh;
  float decay = 1.f;
  uint32_t tmem = 0;
  bool ok = true;
  int done = 0;  // chunks whose products were issued
  for (int i = 0; i < chunks; ++i) {
    const int t0 = first(i);
    const uint32_t par = i & 1;
    if (tid < kQ) {  // warps 0-3: the block's decays and their products
      const int tok = t0 + (int)t;
      const bool l = live(tok);
      const float a = l ? expf(ap[(int64_t)tok * g.log_decay.sl]) : 1.f;
      const float w = l ? (wp ? wp[(int64_t)tok * g.write.sl] : 1.f) : 0.f;
      float head = a, tail = __shfl_down_sync(~0u, a, 1);
      if (lane == 31) tail = 1.f;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float u = __shfl_up_sync(~0u, head, o), d = __shfl_down_sync(~0u, tail, o);
        if ((int)lane >= o) head *= u;
        if ((int)lane + o < 32) tail *= d;
      }
      gate.a[t] = a;
      gate.w[t] = w;
      gate.head[t] = head;
      gate.tail[t] = tail;
      gate.col[t] = (REV ? head : tail) * w;
      if (lane == 31) gate.total[quarter] = head;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_async();
    fence_before();
    ok = __syncthreads_and(ok);
    fence_after();
    if (!ok) break;
    tmem = tslot;
    if constexpr (OUT != kOutNone) {
      if (tid == 0) {
#pragma unroll
        for (uint32_t j = 0; j < COLS / 16; ++j) {
          const uint32_t at = (j >> 2) * kTile + (j & 3) * 32;
          mma_ss(tmem, desc(sq + at, 16), desc(sk + at, 16), idesc(kQ, false, false), j);
        }
#pragma unroll
        for (uint32_t j = 0; j < COLS / 16; ++j) {
          const uint32_t at = (j >> 2) * kTile + (j & 3) * 32;
          mma_ss(tmem + kColO, desc(sq + at, 16), desc(ss + j * 2048, 0), idesc(kRowsTc, false, true), j);
          if constexpr (PRECISE)
            mma_ss(tmem + kColO, desc(sq + at, 16), desc(ss + kBytesS + j * 2048, 0), idesc(kRowsTc, false, true), 1);
        }
        commit(bar_g);
      }
    }
    // products over blocks around this row's and token's own
    float before = 1.f, after = 1.f;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      if (u < quarter) before *= gate.total[u];
      if (u > quarter) after *= gate.total[u];
    }
    const float head = gate.head[t], tail = gate.tail[t], w = gate.w[t];
    const float pt = REV ? tail * after : head * before;
    const float et = (REV ? head * before : tail * after) * w;
    const float all = gate.total[0] * gate.total[1] * gate.total[2] * gate.total[3];
    decay *= all;
    const uint32_t lanes = (quarter * 32) << 16;
    float acc[OUT == kOutNone ? 1 : 32];
    if constexpr (OUT != kOutNone) {
      __syncwarp();
      ok = __all_sync(~0u, wait(bar_g, par));
      done = i + 1;
      fence_after();
      if (ok) {
        tmem_ld32(tmem + lanes + kColO + half * 32, acc);
        ld_wait();
      }
    }
    const float skip = (OUT == kOutY || OUT == kOutDx) && g.d ? g.d[h] : 0.f;
    float oscale = 1.f;
    // U of the gradients: its products are rounded at w_t times their value, as
    // those of dC_h are, with the power of two of w_t left out.  alpha and beta,
    // whose difference is summed, then carry the same roundings and the sum
    // loses them.
    float mant = 1.f;
    if constexpr (REV && OUT == kOutRaw) {
      const int tok = t0 + (int)t;
      const float ws = live(tok) ? g.out_scale.p[b * g.out_scale.sb + tok * g.out_scale.sl + h * g.out_scale.sh] : 1.f;
      const uint32_t bits = __float_as_uint(ws);
      if ((bits >> 23 & 0xff) - 1u < 0xfeu) mant = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
      oscale = 1.f / mant;
    }
    if constexpr (OUT == kOutDx) {
      const int tok = t0 + (int)t;
      oscale = live(tok) ? g.out_scale.p[b * g.out_scale.sb + tok * g.out_scale.sl + h * g.out_scale.sh] : 0.f;
    }
    // the scaled r in two terms, over q; with it P_t (q S0) and the skip term
    if (ok) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const uint32_t at = swz(t, half * 4 + v);
        const uint4 x = *reinterpret_cast<const uint4*>(smem + (sr - sq) + at);
        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = low(u[e]), x1 = high(u[e]);
          split2(et * x0, et * x1, hi[e], lo[e]);
          if constexpr (OUT != kOutNone) {
            float &o0 = acc[8 * v + 2 * e], &o1 = acc[8 * v + 2 * e + 1];
            o0 *= pt;
            o1 *= pt;
            if constexpr (OUT == kOutDx) {
              o0 *= oscale;
              o1 *= oscale;
            }
            o0 = fmaf(skip, x0, o0);
            o1 = fmaf(skip, x1, o1);
          }
        }
        *reinterpret_cast<uint4*>(smem + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(smem + kTile + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      if constexpr (OUT != kOutNone) {
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
          const uint32_t blk = half * 2 + u;
          const bool zero = REV ? blk < quarter : blk > quarter;
          uint32_t hi[16], lo[16];
          if (!zero) {
            float v[32];
            tmem_ld32(tmem + lanes + blk * 32, v);
            ld_wait();
            float row = (REV ? tail : head) * mant;  // times the blocks between
#pragma unroll
            for (uint32_t m = 0; m < 4; ++m)
              if (REV ? (m > quarter && m < blk) : (m > blk && m < quarter)) row *= gate.total[m];
            weigh<REV>(v, gate, blk, blk == quarter, lane, row, mant);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if constexpr (PRECISE) split2(v[2 * e], v[2 * e + 1], hi[e], lo[e]);
              else hi[e] = pack2(v[2 * e], v[2 * e + 1]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) hi[e] = lo[e] = 0;
          }
          tmem_st16(tmem + lanes + blk * 32, hi);
          if constexpr (PRECISE) tmem_st16(tmem + lanes + blk * 32 + 16, lo);
        }
        st_wait();
      }
    }
    fence_async();
    fence_before();
    ok = __syncthreads_and(ok);
    fence_after();
    if (!ok) break;
    if (tid == 0) {
      const uint32_t lead = kHalves == 2 ? kTile : 0;
#pragma unroll
      for (uint32_t j = 0; j < kQ / 16; ++j) {
        const uint64_t a = desc(sk + j * 2048, lead);
        mma_ss(tmem + kColS, a, desc(sq + j * 2048, 0), idesc(kRowsTc, true, true), j);
        mma_ss(tmem + kColS, a, desc(sq + kTile + j * 2048, 0), idesc(kRowsTc, true, true), 1);
      }
      commit(bar_s);
      if constexpr (OUT != kOutNone) {
#pragma unroll
        for (uint32_t j = 0; j < kQ / 16; ++j) {
          const uint32_t a = tmem + (j >> 1) * 32 + (j & 1) * 8;
          mma_ts(tmem + kColO, a, desc(sr + j * 2048, 0), idesc(kRowsTc, false, true), j);
          if constexpr (PRECISE) mma_ts(tmem + kColO, a + 16, desc(sr + j * 2048, 0), idesc(kRowsTc, false, true), 1);
        }
        commit(bar_o);
      }
    }
    __syncwarp();
    ok = __all_sync(~0u, wait(bar_s, par));
    fence_after();
    if (ok) {
      if (i + 1 < chunks) load_kq(first(i + 1));  // q's and k's places are free
      float v[32];
      tmem_ld32(tmem + lanes + kColS + half * 32, v);
      ld_wait();
#pragma unroll
      for (int e = 0; e < 32; ++e) s[e] = fmaf(all, s[e], v[e]);
      if constexpr (OUT != kOutNone) put_state();
    }
    if constexpr (OUT == kOutNone) {
      if (ok && i + 1 < chunks) load_rows(first(i + 1));
    } else {
      ok = __all_sync(~0u, wait(bar_o, par)) && ok;
      fence_after();
      if (ok) {
        if (i + 1 < chunks) load_rows(first(i + 1));
        float v[32];
        tmem_ld32(tmem + lanes + kColO + half * 32, v);
        ld_wait();
        const int tok = t0 + (int)t;
        const uint32_t row = row0 + half * 32;
        if (tok >= t_lo && tok < t_hi && row < g.rows && (OUT != kOutRaw || tok < len)) {
          const bool l = tok < len;
          const int64_t at = (((int64_t)b * g.length + tok) * g.heads + h) * g.rows + row;
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = l ? fmaf(oscale, v[e], acc[e]) : 0.f;
          if constexpr (OUT == kOutRaw) {
            float* o = static_cast<float*>(g.out) + at;
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (row + e < g.rows) *reinterpret_cast<float4*>(o + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          } else {
            T* o = static_cast<T*>(g.out) + at;
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (row + e < g.rows)
                *reinterpret_cast<uint4*>(o + e) = make_uint4(pack2(v[e], v[e + 1]), pack2(v[e + 2], v[e + 3]),
                                                              pack2(v[e + 4], v[e + 5]), pack2(v[e + 6], v[e + 7]));
          }
        }
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (ok) {
    if (g.state_out) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const uint32_t row = row0 + half * 32 + i;
        if (row < g.rows && t < g.cols)
          g.state_out[bh * g.out_bh + seg * g.out_seg + row * g.st_row + t * g.st_col] = s[i];
      }
    }
    if (OUT == kOutNone && row0 == 0 && tid == 0) g.seg_decay[bh * g.nseg + seg] = decay;
  } else if (tid == 0) {
    // a wait ran out: count it, and let what was issued finish (bounded) before the tensor memory goes
    atomicAdd(&g_scan_timeouts, 1u);
    if (done) {
      const uint32_t par = (done - 1) & 1;
      wait(bar_g, par);
      wait(bar_s, par);
      wait(bar_o, par);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tslot), "r"(kTmemCols));
}

template <int COLS, bool REV, int OUT, bool PRECISE>
void launch(const RecArgs& g, uint32_t batch, cudaStream_t st) {
  const uint32_t need = 1024 + 2 * kTile + COLS / 64 * kTile + kTile + COLS * 128 * (PRECISE ? 2 : 1);
  const uint32_t smem = std::max(need, kLeastSmem);
  FHE_CUDA(cudaFuncSetAttribute(k_scan_tc<COLS, REV, OUT, PRECISE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)smem));
  const uint64_t blocks = (uint64_t)((g.rows + kRowsTc - 1) / kRowsTc) * g.heads * g.nseg * batch;
  require(blocks < (1ull << 31), "too many blocks");
  k_scan_tc<COLS, REV, OUT, PRECISE><<<(uint32_t)blocks, kThreadsTc, smem, st>>>(g);
  note_launch();
  FHE_CUDA(cudaGetLastError());
}

}  // namespace

bool scan_tc_ok(const RecArgs& g, bool needs_q) {
  auto aligned = [](const Src& s) {
    return reinterpret_cast<uintptr_t>(s.p) % 16 == 0 && s.sb % 8 == 0 && s.sl % 8 == 0 && s.sh % 8 == 0;
  };
  return g.cols <= 128 && g.rows % 8 == 0 && aligned(g.r) && aligned(g.k) && (!needs_q || aligned(g.q)) &&
         reinterpret_cast<uintptr_t>(g.out) % 16 == 0;
}

void launch_scan_tc(const RecArgs& g, bool rev, int out, uint32_t batch, cudaStream_t st) {
  auto go = [&](auto cols) {
    constexpr int C = decltype(cols)::value;
    if (!rev && out == kOutNone) launch<C, false, kOutNone, false>(g, batch, st);
    else if (!rev && out == kOutY) launch<C, false, kOutY, false>(g, batch, st);
    else if (!rev && out == kOutRaw) launch<C, false, kOutRaw, true>(g, batch, st);
    else if (rev && out == kOutNone) launch<C, true, kOutNone, false>(g, batch, st);
    else if (rev && out == kOutDx) launch<C, true, kOutDx, false>(g, batch, st);
    else if (rev && out == kOutRaw) launch<C, true, kOutRaw, true>(g, batch, st);
    else require(false, "unknown walk", FHE_ERR_INTERNAL);
  };
  if (g.cols <= 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
}

unsigned scan_tc_timeouts() {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, g_scan_timeouts, sizeof(v));
  return v;
}

}  // namespace fhe
