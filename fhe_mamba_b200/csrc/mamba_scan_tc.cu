// Mamba-2 state recurrence for 16-bit activations on the tensor cores
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
// Roundings.  q, k and r are as given; G, O and S accumulate in fp32.
// G o L o w and S0 enter their products as two terms of the activations' type
// (16 bits for bfloat16, 22 for float16: y and dx are off by their own rounding
// alone; with one term their error was 1.1 times that, and a row of 64 tokens
// differed from one of 63).  For the raw sums (OUT kOutRaw) and for E o w o r,
// whose sum is the fp32 state, it is 22 bits and more: three terms of bfloat16
// or two of float16.
// float16's range is brought to the operands by powers of two that follow what a
// chunk holds: each row of G o L o w, the tile of E o w o r and the tile of S0
// enter with their largest value in [2^14, 2^15), so that two terms are off by
// at most 2^-39 of that (half a step of the subnormal numbers) where they do not
// hold 22 bits of their own.  (With the state times 16 and w alone scaled, a
// state's gradient of 1e-6 lost 3 decimal digits, one of 1e-9 all.)
// A NaN or an infinity among the operands would be carried to all tokens of its
// chunk by the products, zeros of L or not: where an output's product is not
// finite, the kernel says so in *bad, and the caller's launches of the fp32 walk,
// idle otherwise, take those outputs over.  (The states between segments hold no
// more NaN than the recurrence's own.)
//
// One CTA walks one (batch, head, tile of rows, segment).  Shared memory holds
// q, k, r and S0's two terms in 128-byte-swizzled tiles of 64 columns; the
// scaled r takes q's place once q has been used, and what tokens read of each
// other fits 1 KB, which keeps two CTAs on an SM, so that one computes while the
// other waits for its loads or its products.  Tensor memory: G (its columns
// become the A operand G o L o w), O (which starts from the scaled q S0^T) and S'
// (before, q times S0's second term).  The state itself stays in registers; the
// element passes take 16 columns at a time, since spilled registers cost more
// than their instructions (what shared memory leaves of the L1 cache is small).
//
// 8 x 4096 bfloat16 tokens of 24 heads x 64, state 128: 240 us (198 with one term
// of G o L o w and S0 and unchecked products), of which memory needs 36 and the
// products about 80 at full rate; a chunk is a chain of products and element
// passes that two CTAs to an SM cover in part (issue slots 45% busy, the tensor
// pipe 29%), and 192 CTAs leave 104 of 148 SMs with one (148 CTAs take 185 us, 296
// take 245).  Loads by tensor maps and stores of 64-byte runs took the load and
// store unit out of that chain (343 us with 16-byte asynchronous copies and
// scattered stores).
//
// A walk that carries no state on (CARRY false: the gradients', a segment of
// one chunk each) leaves S' out and takes 128 rows where there are as many.
#include <algorithm>
#include <atomic>
#include <cuda.h>

#include "launch_count.h"
#include "mamba_ops.h"
#include "mamba_scan.h"

namespace fhe {
namespace {

constexpr uint32_t kQ = 128;            // tokens per chunk (MMA M)
constexpr uint32_t kThreadsTc = 256;
constexpr uint32_t kTile = kQ * 128;    // bytes of a 128 x 64 tile
constexpr uint32_t kTmemCols = 256;     // G 128; O 64 and S' 64, or O 128
constexpr uint32_t kColO = 128, kColS = 192;
// More than a third of an SM's shared memory: at most two CTAs are resident,
// whose tensor memory (2 x 256 columns) fits.
constexpr uint32_t kLeastSmem = 80 * 1024;
// Bound on a wait for loads or products, in polls of a microsecond at most: far
// above what they take.  When one runs out, the CTA counts it, waits (bounded
// again) for what it has in flight, frees its tensor memory and says so: its
// outputs are computed again by the fp32 walk (*bad), a state between segments
// becomes NaN.
constexpr uint32_t kWaitLimit = 1u << 20;
constexpr uint32_t kPoll = 1000;  // ns

__device__ unsigned g_scan_timeouts = 0;
std::atomic<uint32_t> g_wait_limit{kWaitLimit};
std::atomic<uint64_t> g_used_devices{0};  // bit d: device d has run the kernel

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 128-byte-swizzled tiles: 8-row groups 1024 bytes apart; for operands whose
// M or N axis is the contiguous one, the next 64 of it `lead` bytes on.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lead >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kind::f16, operands of type T, fp32 accumulator; a_mn / b_mn: the operand's
// M / N axis is contiguous.
template <class T>
constexpr uint32_t idesc(uint32_t n, bool a_mn, bool b_mn) {
  constexpr uint32_t type = std::is_same_v<T, __half> ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) |
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
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, uint32_t limit) {
  for (uint32_t i = 0; i < limit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity), "r"(kPoll)
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
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
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

// Tensor maps of q, k and r: [batch][token][head or group][column or row], a
// box of 64 columns x 128 tokens.  The tensor's extents end at the row's
// length, columns and rows, past which a box is filled with zeros.
struct Maps {
  CUtensorMap q, k, r;
};
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int col, int head, int tok, int batch,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(col), "r"(head), "r"(tok), "r"(batch), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

template <class T>
__device__ __forceinline__ uint32_t pack2(uint64_t p) {
  float a, b;
  unpair(p, a, b);
  uint32_t v;
  if constexpr (std::is_same_v<T, __half>) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(b), "f"(a));
  return v;
}
template <class T>
__device__ __forceinline__ uint64_t unpack2(uint32_t v) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    return pair(f.x, f.y);
  } else {
    return pair(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
}
// The two terms of T of a pair of floats.
template <class T>
__device__ __forceinline__ void split2(uint64_t p, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(p);
  lo = pack2<T>(fma2(unpack2<T>(hi), pair(-1.f, -1.f), p));
}

// The power of two that brings |v| into [1, 2), 1 for 0, denormals and above 2^100.
__device__ __forceinline__ float scale_of(float v) {
  const uint32_t e = __float_as_uint(v) >> 23 & 0xff;
  return e - 1u < 226u ? __uint_as_float((254u - e) << 23) : 1.f;
}

// The power of two that brings the bits of a |v| into [2^14, 2^15), at most
// 2^`most`; 1 for 0, NaN and infinities.
__device__ __forceinline__ float range_of(uint32_t bits, int most) {
  const int e = (int)(bits >> 23);
  if (bits == 0 || e == 255) return 1.f;
  return __uint_as_float((uint32_t)(127 + min(141 - e, most)) << 23);
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one;
}

// Byte offset of 16-byte word `word` of row `row` in a 128-byte-swizzled tile.
__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t word) { return row * 128 + ((word ^ (row & 7)) << 4); }

// What a chunk's threads read of each other's tokens, with the barriers: 1 KB,
// which is what two CTAs' tiles leave of an SM's shared memory.
template <bool REV>
struct Small {
  float cols[96];   // column factor for rows of other blocks of 32: tail (reversed: head) times w
  float col8[kQ];   // and for rows of other blocks of 8 in its block of 32
  float total[4];   // product over each block of 32
  uint32_t state[8];  // bits of the largest |S0| of each warp (float16)
  uint64_t bars[5];  // G and q S0, S', O; k and q have arrived, r has
  uint32_t tslot;
  uint32_t issued;  // thread 0's, by index of the barrier: whether anything was issued, and the parity of how often
  // no row lies beyond the last (reversed: before the first) block of 32
  __device__ __forceinline__ float* col(uint32_t blk) { return cols + (blk - (REV ? 1u : 0u)) * 32; }
};
constexpr uint32_t kSmall = 1024;
static_assert(sizeof(Small<false>) <= kSmall, "shared memory");

// A token's decay and write, and the products of decays over its block of 32:
// up to and with the token, and after it.
struct Token {
  float a, w, head, tail;
};

// All warps, one token per thread; those of `put` (four) leave the chunk's column factors.
template <bool REV>
__device__ __forceinline__ Token make_token(Small<REV>& g, uint32_t t, uint32_t lane, float a, float w, bool put) {
  const float after = __shfl_down_sync(~0u, a, 1);
  const int in = lane & 7;
  float head = a, head8 = a, tail = lane == 31 ? 1.f : after, tail8 = in == 7 ? 1.f : after;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float u = __shfl_up_sync(~0u, head, o), d = __shfl_down_sync(~0u, tail, o);
    if ((int)lane >= o) head *= u;
    if ((int)lane + o < 32) tail *= d;
    if (o < 8) {
      const float u8 = __shfl_up_sync(~0u, head8, o), d8 = __shfl_down_sync(~0u, tail8, o);
      if (in >= o) head8 *= u8;
      if (in + o < 8) tail8 *= d8;
    }
  }
  if (put) {
    const uint32_t blk = t >> 5;
    if (REV ? blk > 0 : blk < 3) g.col(blk)[lane] = (REV ? head : tail) * w;
    g.col8[t] = (REV ? head8 : tail8) * w;
    if (lane == 31) g.total[blk] = head;
  }
  return Token{a, w, head, tail};
}

// A row's factors within its own block of 32, times `scale`: `own` for the
// columns of its block of 8 (zero off the triangle), `row` for the columns of
// the other blocks of 8, times their col8.
struct OwnBlock {
  float own[8], row[4];
};
template <bool REV>
__device__ __forceinline__ OwnBlock own_block(const Token& g, uint32_t lane, float scale) {
  OwnBlock o;
  const int sub = lane >> 3, in = lane & 7;
  float a[8], w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = __shfl_sync(~0u, g.a, i, 8);
    w[i] = __shfl_sync(~0u, g.w, i, 8);
  }
  float p = scale, all = 1.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = REV ? j : 7 - j;
    // scale times the product of a over (i, in], or over (in, i]
    if constexpr (REV) p = i > in ? p * a[i] : scale;
    else if (i < 7) p = i < in ? p * a[i + 1] : scale;
    o.own[i] = (REV ? i >= in : i <= in) ? p * w[i] : 0.f;
    all *= a[i];
  }
  const float edge = REV ? p : p * a[0];  // to the end (the start, with the token) of its block of 8
  float tot[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) tot[j] = __shfl_sync(~0u, all, 8 * j);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float r = edge;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (REV ? (m > sub && m < j) : (m > j && m < sub)) r *= tot[m];
    o.row[j] = (REV ? j > sub : j < sub) ? r : 0.f;
  }
  return o;
}

// 16 columns of G o L o w for one row, in place: columns of another block of
// 32, and (from group j of 8 on) of the row's own.
__device__ __forceinline__ void weigh(float (&v)[16], const float* col, float row) {
  const uint64_t rr = pair(row, row);
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(col + i);
    unpair(mul2(pair(v[i], v[i + 1]), mul2(rr, c.x)), v[i], v[i + 1]);
    unpair(mul2(pair(v[i + 2], v[i + 3]), mul2(rr, c.y)), v[i + 2], v[i + 3]);
  }
}
__device__ __forceinline__ void weigh_own(float (&v)[16], const float* col8, const OwnBlock& o, uint32_t lane, int j0) {
  const int sub = lane >> 3;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint64_t rr = pair(o.row[j0 + j], o.row[j0 + j]);
    const bool mine = sub == j0 + j;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(col8 + 8 * j + i);
      float f[4];
      unpair(mul2(rr, c.x), f[0], f[1]);
      unpair(mul2(rr, c.y), f[2], f[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = mine ? o.own[i + e] : f[e];
      float* x = v + 8 * j + i;
      unpair(mul2(pair(x[0], x[1]), pair(f[0], f[1])), x[0], x[1]);
      unpair(mul2(pair(x[2], x[3]), pair(f[2], f[3])), x[2], x[3]);
    }
  }
}

// COLS: columns held, 64 or 128 (those past g.cols are zeros); ROWS: rows per
// CTA, 64 or 128 (128 only without CARRY).
template <class T, int COLS, int ROWS, bool REV, int OUT, bool CARRY>
__global__ void __launch_bounds__(kThreadsTc, 2) k_scan_tc(const RecArgs g, const __grid_constant__ Maps maps) {
  static_assert((CARRY ? OUT != kOutRaw : OUT != kOutNone) && (ROWS == 64 || OUT == kOutRaw), "shapes");
  constexpr uint32_t kHalves = COLS / 64, kRowTiles = ROWS / 64;
  constexpr uint32_t kBytesQ = CARRY ? 2 * kTile : kHalves * kTile;  // q, then the scaled r (two terms)
  constexpr uint32_t kBytesK = kHalves * kTile;
  constexpr uint32_t kBytesR = kRowTiles * kTile;
  constexpr uint32_t kTileS = COLS * 128, kBytesS = kRowTiles * kTileS;
  constexpr bool kThird = CARRY && !std::is_same_v<T, __half>;  // a third term of the scaled r, in S0's place
  // The raw sums' third terms: of S0 in r's place, and of the weighted G as an
  // operand in q's and k's (dwrite of 4 x 2048 bfloat16 tokens 4e-7 to 6e-7 off,
  // 2.4e-6 with two; 69 us a pass)
  constexpr bool kThirds = OUT == kOutRaw && !std::is_same_v<T, __half>;
  // One product gives q times both terms of S0, side by side: the second's takes
  // the place of S', not needed yet.
  constexpr bool kPair = OUT != kOutNone && ROWS == 64 && !kThirds;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Small<REV>& gate = *reinterpret_cast<Small<REV>*>(smem_raw);
  uint8_t* smem = smem_raw + kSmall;  // the tiles
  const uint32_t sq = smem_u32(smem), sk = sq + kBytesQ, sr = sk + kBytesK;
  const uint32_t ss = sr + kBytesR;  // S0, two terms
  const uint32_t bar_g = smem_u32(&gate.bars[0]), bar_s = bar_g + 8, bar_o = bar_g + 16, bar_kq = bar_g + 24,
                 bar_r = bar_g + 32;

  const uint32_t tiles = (g.rows + ROWS - 1) / ROWS;
  uint32_t id = blockIdx.x;
  const uint32_t row0 = id % tiles * ROWS;
  id /= tiles;
  const uint32_t h = id % g.heads;
  id /= g.heads;
  const uint32_t seg = id % g.nseg, b = id / g.nseg;
  const int64_t bh = (int64_t)b * g.heads + h;
  const int len = clamp_length(g.lengths, b, g.length);
  const int t_lo = seg * g.seglen, t_hi = min(t_lo + (int)g.seglen, (int)g.length);
  const int t_end = min(t_hi, len);  // live tokens: [t_lo, t_end)
  const int chunks = (t_hi - t_lo + (int)kQ - 1) / (int)kQ;

  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t quarter = warp & 3, half = warp >> 2;
  const uint32_t t = quarter * 32 + lane;  // this thread's token, and column of S
  constexpr bool kHalf = std::is_same_v<T, __half>;
  float sigma = 1.f;  // float16: scale of S0 in shared memory
  // A sum of 0 times every product: NaN once one is not finite.
  auto report = [&](uint64_t poison) {
    float a, c;
    unpair(poison, a, c);
    if (!(a == 0.f && c == 0.f)) *g.bad = 1;
  };

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&gate.tslot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 0) {
    gate.issued = 0;
    for (int i = 0; i < 5; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar_g + 8 * i));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }

  auto note = [&](int bar) { gate.issued = (gate.issued ^ 1u << bar) | 256u << bar; };
  auto first = [&](int i) { return t_lo + (int)kQ * (REV ? chunks - 1 - i : i); };
  // One thread: the boxes of a chunk.
  auto load_rows = [&](int t0) {
    expect(bar_r, kBytesR);
    note(4);
#pragma unroll
    for (uint32_t j = 0; j < kRowTiles; ++j) load_box(sr + j * kTile, &maps.r, row0 + 64 * j, h / g.r.share, t0, b, bar_r);
  };
  auto load_kq = [&](int t0) {
    expect(bar_kq, kBytesK * (OUT != kOutNone ? 2 : 1));
    note(3);
#pragma unroll
    for (uint32_t j = 0; j < kHalves; ++j) {
      load_box(sk + j * kTile, &maps.k, 64 * j, h / g.k.share, t0, b, bar_kq);
      if constexpr (OUT != kOutNone) load_box(sq + j * kTile, &maps.q, 64 * j, h / g.q.share, t0, b, bar_kq);
    }
  };
  // Tokens past the sequence's end that lie within the row were loaded too:
  // this thread's words of them become zeros.
  auto clear = [&](uint32_t tile, uint32_t count) {
    for (uint32_t j = 0; j < count; ++j)
#pragma unroll
      for (uint32_t v = 0; v < 4; ++v)
        *reinterpret_cast<uint4*>(smem + (tile - sq) + j * kTile + swz(t, half * 4 + v)) = make_uint4(0, 0, 0, 0);
  };
  if (tid == 0) {
    load_kq(first(0));
    if constexpr (!kThirds) load_rows(first(0));
  }

  const float* wp = g.write.p ? g.write.p + (int64_t)b * g.write.sb + (int64_t)h * g.write.sh : nullptr;
  const float* ap = g.log_decay.p + (int64_t)b * g.log_decay.sb + (int64_t)h * g.log_decay.sh;
  float next_a = 0.f, next_w = 0.f;  // the gates of the chunk to come
  auto load_gates = [&](int t0) {
    const int tok = t0 + (int)t;
    const bool l = tok < t_end;
    next_a = l ? ap[(int64_t)tok * g.log_decay.sl] : 0.f;
    next_w = l ? (wp ? wp[(int64_t)tok * g.write.sl] : 1.f) : 0.f;
  };
  load_gates(first(0));
  float row_w = 1.f;  // without CARRY: w of this thread's token, for its row scale
  if constexpr (OUT == kOutDx || (REV && OUT == kOutRaw)) {
    const int tok = first(0) + (int)t;
    if (tok < t_end) row_w = g.out_scale.p[b * g.out_scale.sb + tok * g.out_scale.sl + h * g.out_scale.sh];
  }
  const float skip = (OUT == kOutY || OUT == kOutDx) && g.d ? g.d[h] : 0.f;

  // The state: column t of 32 rows, in pairs; in shared memory it is the B
  // operand [column][row].
  uint64_t s[16];
  [[maybe_unused]] auto put_state = [&](uint32_t piece) {
    if (t >= (uint32_t)COLS) return;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t x = kHalf ? mul2(s[4 * v + e], pair(sigma, sigma)) : s[4 * v + e];
        split2<T>(x, hi[e], lo[e]);
      }
      const uint32_t at = ss - sq + (piece >> 1) * kTileS + swz(t, (piece & 1) * 4 + v);
      *reinterpret_cast<uint4*>(smem + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(smem + at + kBytesS) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  };
  // float16: the tile's scale from its largest value; a barrier in between
  [[maybe_unused]] auto find_sigma = [&](uint32_t bits) {
    bits = __reduce_max_sync(~0u, bits);
    if (lane == 0) gate.state[warp] = bits;
    __syncthreads();
    bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) bits = max(bits, gate.state[i]);
    sigma = range_of(bits, 126);
  };
  [[maybe_unused]] auto state_bits = [&] {
    uint32_t bits = 0;
    if (t < g.cols) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float a, c;
        unpair(s[i], a, c);
        bits = max(bits, __float_as_uint(fmaxf(fabsf(a), fabsf(c))));
      }
    }
    return bits;
  };
  if constexpr (OUT == kOutRaw) {
    // rows run along memory here (st_row 1): a warp takes a column's 128 rows
    // at a time, four to a lane
    const float* in = g.state_in + bh * g.in_bh + seg * g.in_seg;
    constexpr uint32_t kLoads = COLS * ROWS / 4 / kThreadsTc, per = ROWS / 4;  // groups of four rows
    float4 own[kHalf ? kLoads : 1];  // (float16: all of them, for their scale)
    auto fetch = [&](uint32_t j) {
      const uint32_t e = j * kThreadsTc + tid, c = e / per, row = row0 + e % per * 4;
      return c < g.cols && row < g.rows ? *reinterpret_cast<const float4*>(in + (int64_t)c * g.st_col + row)
                                        : make_float4(0, 0, 0, 0);
    };
    if constexpr (kHalf) {
      uint32_t bits = 0;
#pragma unroll
      for (uint32_t j = 0; j < kLoads; ++j) {
        own[j] = fetch(j);
        bits = max(bits, __float_as_uint(fmaxf(fmaxf(fabsf(own[j].x), fabsf(own[j].y)),
                                               fmaxf(fabsf(own[j].z), fabsf(own[j].w)))));
      }
      find_sigma(bits);
    }
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
      const uint32_t e = j * kThreadsTc + tid, c = e / per, n = e % per * 4;
      const float4 x = kHalf ? own[kHalf ? j : 0] : fetch(j);
      uint2 hi, lo;
      split2<T>(pair(sigma * x.x, sigma * x.y), hi.x, lo.x);
      split2<T>(pair(sigma * x.z, sigma * x.w), hi.y, lo.y);
      const uint32_t at = ss - sq + (n >> 6) * kTileS + swz(c, n >> 3 & 7) + (n & 4) * 2;
      *reinterpret_cast<uint2*>(smem + at) = hi;
      *reinterpret_cast<uint2*>(smem + at + kBytesS) = lo;
      if constexpr (kThirds) {
        const uint64_t m1 = pair(-1.f, -1.f);
        *reinterpret_cast<uint2*>(smem + at - (ss - sr)) =
            make_uint2(pack2<T>(fma2(unpack2<T>(lo.x), m1, fma2(unpack2<T>(hi.x), m1, pair(x.x, x.y)))),
                       pack2<T>(fma2(unpack2<T>(lo.y), m1, fma2(unpack2<T>(hi.y), m1, pair(x.z, x.w)))));
      }
    }
  } else {
    const float* in = OUT != kOutNone && g.state_in && t < g.cols
                          ? g.state_in + bh * g.in_bh + seg * g.in_seg + (int64_t)t * g.st_col : nullptr;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t row = row0 + half * 32 + 2 * i;
      s[i] = pair(in && row < g.rows ? in[row * g.st_row] : 0.f,
                  in && row + 1 < g.rows ? in[(row + 1) * g.st_row] : 0.f);
    }
    if constexpr (OUT != kOutNone) {
      if constexpr (kHalf) find_sigma(state_bits());
      put_state(half);
    }
  }

  float decay = 1.f;
  uint32_t tmem = 0;
  const uint32_t lanes = (quarter * 32) << 16;
  bool ok = true;
  for (int i = 0; i < chunks; ++i) {
    const int t0 = first(i), tok = t0 + (int)t;
    const bool live = tok < t_end;
    const uint32_t par = i & 1;
    // (column factors by warps 4-7: warp 0 has the products to issue)
    const Token me = make_token<REV>(gate, t, lane, expf(next_a), next_w, half == 1);
    // Row scale of this token's products: w of dx; for U of the gradients the
    // mantissa of w, so that its products are rounded at w_t times their value
    // as those of dC_h are, up to a power of two.  alpha and beta, whose
    // difference is summed, then carry the same roundings and the sum loses
    // them.  `up` undoes what the row scale took too much.
    float rho = 1.f, up = 1.f;
    if constexpr (OUT == kOutDx || (REV && OUT == kOutRaw)) {
      const float w = row_w;
      rho = OUT == kOutRaw ? w * scale_of(w) : w;
      if constexpr (OUT == kOutRaw) {
        if (fabsf(rho) < 1.f) rho = 1.f;  // 0 or denormal
        up = 1.f / rho;
      }
    }
    if (i > 0) {  // (the barriers are initialised before the first)
      ok = __all_sync(~0u, wait(bar_kq, par, g.wait_limit)) && ok;
      if (!live && t_end < t_hi) {
        clear(sk, kHalves);
        if constexpr (OUT != kOutNone) clear(sq, kHalves);
      }
    }
    fence_async();
    fence_before();
    ok = __syncthreads_and(ok);
    fence_after();
    if (!ok) break;
    if (i == 0) {
      ok = __all_sync(~0u, wait(bar_kq, par, g.wait_limit));
      if (!live && t_end < t_hi) {
        clear(sk, kHalves);
        if constexpr (OUT != kOutNone) clear(sq, kHalves);
      }
      fence_async();
      ok = __syncthreads_and(ok);
      if (!ok) break;
    }
    tmem = gate.tslot;
    if (OUT != kOutNone && warp == 0) {
      if (elect_one()) {
#pragma unroll
        for (uint32_t j = 0; j < COLS / 16; ++j) {
          const uint32_t at = (j >> 2) * kTile + (j & 3) * 32;
          mma_ss(tmem, desc(sq + at, 16), desc(sk + at, 16), idesc<T>(kQ, false, false), j);
        }
#pragma unroll
        for (uint32_t j = 0; j < COLS / 16; ++j) {
          const uint32_t at = (j >> 2) * kTile + (j & 3) * 32;
          if constexpr (kPair) {
            mma_ss(tmem + kColO, desc(sq + at, 16), desc(ss + j * 2048, kTileS), idesc<T>(128, false, true), j);
          } else {
            mma_ss(tmem + kColO, desc(sq + at, 16), desc(ss + j * 2048, kTileS), idesc<T>(ROWS, false, true), j);
            mma_ss(tmem + kColO, desc(sq + at, 16), desc(ss + kBytesS + j * 2048, kTileS), idesc<T>(ROWS, false, true), 1);
          }
          if constexpr (kThirds)
            mma_ss(tmem + kColO, desc(sq + at, 16), desc(sr + j * 2048, kTileS), idesc<T>(ROWS, false, true), 1);
        }
        commit(bar_g);
      }
      __syncwarp();
      if (tid == 0) note(0);
    }
    if (i + 1 < chunks) load_gates(first(i + 1));
    // products over the blocks around this row's own
    float before = 1.f, after = 1.f;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      if (u < quarter) before *= gate.total[u];
      if (u > quarter) after *= gate.total[u];
    }
    const float pt = (REV ? me.tail * after : me.head * before) * rho;
    float et = (REV ? me.head * before : me.tail * after) * me.w;
    float keep = skip / up;  // the skip term in the products' scale
    const float all = gate.total[0] * gate.total[1] * gate.total[2] * gate.total[3];
    decay *= all;
    const bool owner = half == (quarter == 1 || quarter == 2 ? 1u : 0u);  // half 0: blocks 0 and 3, half 1: 1 and 2
    OwnBlock ob;
    if constexpr (OUT != kOutNone) {
      if (owner) ob = own_block<REV>(me, lane, rho);
      ok = __all_sync(~0u, wait(bar_g, par, g.wait_limit));
      fence_after();
    }
    if constexpr (kThirds) {
      if (ok && tid == 0) load_rows(t0);
      __syncwarp();
    }
    [[maybe_unused]] float largest = 0.f;  // of this row's products in its two blocks (float16)
    if constexpr (OUT != kOutNone) {
      if (ok) {
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
          const uint32_t blk = half ? 1 + u : 3 * u;
          const bool zero = REV ? blk < quarter : blk > quarter;
          float row = (REV ? me.tail : me.head) * rho;  // times the blocks between
#pragma unroll
          for (uint32_t m = 0; m < 4; ++m)
            if (REV ? (m > quarter && m < blk) : (m > blk && m < quarter)) row *= gate.total[m];
#pragma unroll
          for (uint32_t n = 0; n < 2; ++n) {  // 16 columns: their first terms, then their second
            const uint32_t at = tmem + lanes + blk * 32 + n * 16;
            uint32_t x[16], third[8];
            if (!zero) {
              float v[16];
              tmem_ld16(at, v);
              ld_wait();
              if (blk == quarter) weigh_own(v, &gate.col8[blk * 32 + n * 16], ob, lane, 2 * n);
              else weigh(v, gate.col(blk) + n * 16, row);
              if constexpr (kHalf) {  // as they are; the row's scale is found first
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  largest = fmaxf(largest, fabsf(v[e]));
                  x[e] = __float_as_uint(v[e]);
                }
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const uint64_t p = pair(v[2 * e], v[2 * e + 1]);
                  split2<T>(p, x[e], x[8 + e]);
                  if constexpr (kThirds)
                    third[e] =
                        pack2<T>(fma2(unpack2<T>(x[8 + e]), pair(-1.f, -1.f), fma2(unpack2<T>(x[e]), pair(-1.f, -1.f), p)));
                }
              }
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = x[8 + e] = third[e] = 0;
            }
            if constexpr (kThirds) {
#pragma unroll
              for (int e = 0; e < 2; ++e)
                *reinterpret_cast<uint4*>(smem + (blk >> 1) * kTile + swz(t, (blk & 1) * 4 + n * 2 + e)) =
                    make_uint4(third[4 * e], third[4 * e + 1], third[4 * e + 2], third[4 * e + 3]);
            }
            tmem_st16(at, x);
          }
        }
      }
    }
    ok = __all_sync(~0u, wait(bar_r, par, g.wait_limit)) && ok;
    if (!live && t_end < t_hi) clear(sr, kRowTiles);
    float back = 1.f, scale = 1.f;  // float16: undoes the scale of E o w o r; S0's to the row's
    if constexpr (kHalf) {
      // The scales of this row's products and of the tile of E o w o r: the row's
      // other half and the other warps are told over S0's place, which is free.
      uint32_t* told = reinterpret_cast<uint32_t*>(smem + (ss - sq));
      if (OUT != kOutNone) told[half * kQ + t] = __float_as_uint(largest);
      if constexpr (CARRY) {
        __half2 most = __half2half2(__ushort_as_half(0));
#pragma unroll
        for (uint32_t v = 0; v < 4; ++v) {
          const uint4 q4 = *reinterpret_cast<const uint4*>(smem + (sr - sq) + swz(t, half * 4 + v));
          const uint32_t q[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
          for (int f = 0; f < 4; ++f) most = __hmax2(most, __habs2(*reinterpret_cast<const __half2*>(&q[f])));
        }
        const float2 m = __half22float2(most);
        const uint32_t bits = __reduce_max_sync(~0u, __float_as_uint(fabsf(et) * fmaxf(m.x, m.y)));
        if (lane == 0) told[2 * kQ + warp] = bits;
      }
      __syncthreads();
      if constexpr (CARRY) {
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) bits = max(bits, told[2 * kQ + i]);
        const float up_r = range_of(bits, 100);
        et *= up_r;
        back = 1.f / up_r;
      }
      if constexpr (OUT != kOutNone) {
        // (at most 2^60: the row's other terms, of the state, stay in fp32's range)
        const float f = range_of(max(__float_as_uint(largest), told[(half ^ 1u) * kQ + t]), 60);
        scale = f / sigma;
        keep *= f;
        up /= f;
        if (ok) {
          st_wait();
#pragma unroll
          for (uint32_t u = 0; u < 2; ++u) {
            const uint32_t blk = half ? 1 + u : 3 * u;
            if (REV ? blk < quarter : blk > quarter) continue;
#pragma unroll
            for (uint32_t n = 0; n < 2; ++n) {
              const uint32_t at = tmem + lanes + blk * 32 + n * 16;
              float v[16];
              uint32_t x[16];
              tmem_ld16(at, v);
              ld_wait();
#pragma unroll
              for (int e = 0; e < 8; ++e) split2<T>(mul2(pair(v[2 * e], v[2 * e + 1]), pair(f, f)), x[e], x[8 + e]);
              tmem_st16(at, x);
            }
          }
        }
      }
    }
    if (ok) {
      // O starts from P_t (q S0) and the skip term; the scaled r, in two terms, goes over q
#pragma unroll
      for (uint32_t u = 0; u < 2 * kRowTiles; ++u) {
        const uint32_t part = half * 2 * kRowTiles + u;  // 16 rows
        float v[16];
        if constexpr (OUT != kOutNone) {
          tmem_ld16(tmem + lanes + kColO + part * 16, v);
          if constexpr (kPair) {
            float low[16];
            tmem_ld16(tmem + lanes + kColS + part * 16, low);
            ld_wait();
#pragma unroll
            for (int e = 0; e < 16; e += 2) unpair(add2(pair(v[e], v[e + 1]), pair(low[e], low[e + 1])), v[e], v[e + 1]);
          } else {
            ld_wait();
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t at = (part >> 2) * kTile + swz(t, (part & 3) * 2 + e);
          uint32_t x[4] = {0, 0, 0, 0};
          if constexpr (CARRY || OUT == kOutY || OUT == kOutDx) {
            const uint4 q4 = *reinterpret_cast<const uint4*>(smem + (sr - sq) + at);
            x[0] = q4.x, x[1] = q4.y, x[2] = q4.z, x[3] = q4.w;
          }
          uint32_t hi[4], lo[4], third[4];
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const uint64_t xx = unpack2<T>(x[f]);
            if constexpr (CARRY) {
              const uint64_t scaled = mul2(pair(et, et), xx);
              split2<T>(scaled, hi[f], lo[f]);
              if constexpr (kThird)
                third[f] = pack2<T>(fma2(unpack2<T>(lo[f]), pair(-1.f, -1.f),
                                         fma2(unpack2<T>(hi[f]), pair(-1.f, -1.f), scaled)));
            }
            if constexpr (OUT != kOutNone) {
              float *o = v + 8 * e + 2 * f;
              uint64_t a = mul2(pair(pt, pt), pair(o[0], o[1]));
              if constexpr (kHalf) a = mul2(pair(scale, scale), a);
              if constexpr (OUT == kOutY || OUT == kOutDx) a = fma2(pair(keep, keep), xx, a);
              unpair(a, o[0], o[1]);
            }
          }
          if constexpr (CARRY) {
            *reinterpret_cast<uint4*>(smem + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(smem + kTile + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            if constexpr (kThird)
              *reinterpret_cast<uint4*>(smem + (ss - sq) + at) = make_uint4(third[0], third[1], third[2], third[3]);
          }
        }
        if constexpr (OUT != kOutNone) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(v[e]);
          tmem_st16(tmem + lanes + kColO + part * 16, w);
        }
      }
      if constexpr (OUT != kOutNone) st_wait();
    }
    fence_async();
    fence_before();
    ok = __syncthreads_and(ok);
    fence_after();
    if (!ok) break;
    if (warp == 0) {
      if (elect_one()) {
        if constexpr (CARRY) {
          const uint32_t lead = kHalves == 2 ? kTile : 0;
#pragma unroll
          for (uint32_t j = 0; j < kQ / 16; ++j) {
            const uint64_t a = desc(sk + j * 2048, lead);
            mma_ss(tmem + kColS, a, desc(sq + j * 2048, 0), idesc<T>(64, true, true), j);
            mma_ss(tmem + kColS, a, desc(sq + kTile + j * 2048, 0), idesc<T>(64, true, true), 1);
            if constexpr (kThird) mma_ss(tmem + kColS, a, desc(ss + j * 2048, 0), idesc<T>(64, true, true), 1);
          }
          commit(bar_s);
        }
        if constexpr (OUT != kOutNone) {
#pragma unroll
          for (uint32_t j = 0; j < kQ / 16; ++j) {
            const uint32_t a = tmem + j * 16;
            mma_ts(tmem + kColO, a, desc(sr + j * 2048, kTile), idesc<T>(ROWS, false, true), 1);
            mma_ts(tmem + kColO, a + 8, desc(sr + j * 2048, kTile), idesc<T>(ROWS, false, true), 1);
            if constexpr (kThirds)
              mma_ss(tmem + kColO, desc(sq + (j >> 2) * kTile + (j & 3) * 32, 16), desc(sr + j * 2048, kTile),
                     idesc<T>(ROWS, false, true), 1);
          }
          commit(bar_o);
        }
      }
      __syncwarp();
      if (CARRY && tid == 0) note(1);
      if (OUT != kOutNone && tid == 0) note(2);
    }
    if constexpr (CARRY) {
      ok = __all_sync(~0u, wait(bar_s, par, g.wait_limit));
      fence_after();
      if (ok) {
        if (i + 1 < chunks && tid == 0) load_kq(first(i + 1));  // q's and k's places are free
        __syncwarp();
        float v[32];
        tmem_ld32(tmem + lanes + kColS + half * 32, v);
        ld_wait();
        [[maybe_unused]] uint64_t poison = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          uint64_t x = pair(v[2 * e], v[2 * e + 1]);
          if constexpr (kHalf) x = mul2(x, pair(back, back));
          s[e] = fma2(pair(all, all), s[e], x);
          if constexpr (OUT != kOutNone) poison = fma2(s[e], 0, poison);
        }
        if constexpr (OUT != kOutNone) {
          report(poison);
          if (!kHalf && i + 1 < chunks) put_state(half);
        }
      }
    }
    if constexpr (kHalf && CARRY && OUT != kOutNone) {
      if (i + 1 < chunks) {  // the same for all threads
        find_sigma(state_bits());
        if (ok) put_state(half);
      }
    }
    if constexpr (OUT == kOutNone) {
      if (ok && i + 1 < chunks && tid == 0) load_rows(first(i + 1));
    } else {
      ok = __all_sync(~0u, wait(bar_o, par, g.wait_limit)) && ok;
      fence_after();
      if (ok) {
        if (i + 1 < chunks && tid == 0) load_rows(first(i + 1));
        __syncwarp();
#pragma unroll
        for (uint32_t u = 0; u < kRowTiles; ++u) {
          const uint32_t piece = half * kRowTiles + u, row = row0 + piece * 32;
          auto load = [&](uint32_t n, float (&v)[16]) {  // 16 of its rows
            tmem_ld16(tmem + lanes + kColO + piece * 32 + n * 16, v);
            ld_wait();
            uint64_t poison = 0;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const uint64_t x = pair(v[e], v[e + 1]);
              poison = fma2(x, 0, poison);
              if constexpr (kHalf || (OUT == kOutRaw && REV)) unpair(mul2(x, pair(up, up)), v[e], v[e + 1]);
            }
            report(poison);
          };
          // Four lanes hold words of four tokens each; transposed among them,
          // every store covers whole 64-byte runs of eight tokens.
          auto transpose = [&](uint32_t (&x)[4][4]) {
#pragma unroll
            for (int d = 1; d < 4; d *= 2) {
              const bool up = lane & d;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (e & d) continue;
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                  const uint32_t send = up ? x[e][f] : x[e + d][f];
                  const uint32_t got = __shfl_xor_sync(~0u, send, d);
                  if (up) x[e][f] = got;
                  else x[e + d][f] = got;
                }
              }
            }
          };  // x[e]: word lane & 3 of the token 4 (lane / 4) + e of the warp's 32
          if constexpr (OUT == kOutRaw) {
#pragma unroll
            for (int part = 0; part < 2; ++part) {  // 16 rows: four words of four
              float v[16];
              load(part, v);
              uint32_t x[4][4];
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e / 4][e % 4] = __float_as_uint(v[e]);
              transpose(x);
              const uint32_t col = row + 16 * part + 4 * (lane & 3);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int tk = t0 + (int)(quarter * 32 + (lane & ~3u) + e);
                if (tk < t_end && col < g.rows)
                  *reinterpret_cast<uint4*>(static_cast<float*>(g.out) +
                                            (((int64_t)b * g.length + tk) * g.heads + h) * g.rows + col) =
                      make_uint4(x[e][0], x[e][1], x[e][2], x[e][3]);
              }
            }
          }
          if constexpr (OUT != kOutRaw) {
            uint32_t x[4][4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              float v[16];
              load(n, v);
#pragma unroll
              for (int e = 0; e < 8; ++e) x[2 * n + e / 4][e % 4] = live ? pack2<T>(pair(v[2 * e], v[2 * e + 1])) : 0u;
            }
            transpose(x);
            const uint32_t col = row + 8 * (lane & 3);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int tk = t0 + (int)(quarter * 32 + (lane & ~3u) + e);
              if (tk < t_hi && col < g.rows)
                *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + (((int64_t)b * g.length + tk) * g.heads + h) * g.rows +
                                          col) = make_uint4(x[e][0], x[e][1], x[e][2], x[e][3]);
            }
          }
        }
      }
    }
  }
  if (CARRY && g.state_out && t < g.cols && (ok || OUT == kOutNone)) {
    float* o = g.state_out + bh * g.out_bh + seg * g.out_seg + (int64_t)t * g.st_col;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t row = row0 + half * 32 + 2 * i;
      float a, c;
      unpair(s[i], a, c);
      if (row < g.rows) o[row * g.st_row] = ok ? a : NAN;
      if (row + 1 < g.rows) o[(row + 1) * g.st_row] = ok ? c : NAN;
    }
  }
  if (OUT == kOutNone && row0 == 0 && tid == 0) g.seg_decay[bh * g.nseg + seg] = decay;
  if (!ok && tid == 0) {
    atomicAdd(&g_scan_timeouts, 1u);
    if (OUT != kOutNone) *g.bad = 1;
    for (int i = 0; i < 5; ++i)  // what is in flight ends before its memory goes
      if (gate.issued >> (8 + i) & 1) wait(bar_g + 8 * i, (gate.issued >> i & 1) ^ 1, kWaitLimit);
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(gate.tslot), "r"(kTmemCols));
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encoder() {
  static const Encode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<Encode>(p);
  }();
  return fn;
}

// The map of one operand; false if its layout has none.
bool make_map(CUtensorMap& m, const Src& s, uint32_t width, const RecArgs& g, uint32_t batch, bool half) {
  const Encode fn = encoder();
  if (!fn) return false;
  const uint64_t dims[4] = {width, g.heads / s.share, g.length, batch};
  const int64_t at[3] = {s.sh, s.sl, s.sb};
  uint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    if (dims[i + 1] > 1 && (at[i] <= 0 || at[i] % 8 != 0)) return false;
    strides[i] = dims[i + 1] > 1 ? (uint64_t)at[i] * 2 : 16;  // an axis of one element never moves
  }
  const cuuint64_t d[4] = {dims[0], dims[1], dims[2], dims[3]}, st[3] = {strides[0], strides[1], strides[2]};
  const cuuint32_t box[4] = {64, 1, kQ, 1}, step[4] = {1, 1, 1, 1};
  return reinterpret_cast<uintptr_t>(s.p) % 16 == 0 &&
         fn(&m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(s.p), d, st, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int COLS, int ROWS, bool REV, int OUT, bool CARRY>
void launch(const RecArgs& g, const Maps& maps, uint32_t batch, cudaStream_t st) {
  const uint32_t need = kSmall + (CARRY ? 2 : COLS / 64) * kTile + COLS / 64 * kTile + ROWS / 64 * kTile +
                        (OUT == kOutNone ? kTile : COLS * 128u * (ROWS / 64) * 2);
  const uint32_t smem = std::max(need, kLeastSmem);
  auto* kernel = k_scan_tc<T, COLS, ROWS, REV, OUT, CARRY>;
  FHE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  FHE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  const uint64_t blocks = (uint64_t)((g.rows + ROWS - 1) / ROWS) * g.heads * g.nseg * batch;
  require(blocks < (1ull << 31), "too many blocks");
  int device = 0;
  FHE_CUDA(cudaGetDevice(&device));
  g_used_devices.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
  kernel<<<(uint32_t)blocks, kThreadsTc, smem, st>>>(g, maps);
  note_launch();
  FHE_CUDA(cudaGetLastError());
}

}  // namespace

template <class T>
bool launch_scan_tc(RecArgs g, bool rev, int out, uint32_t batch, cudaStream_t st) {
  g.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
  constexpr bool kHalf = std::is_same_v<T, __half>;
  Maps maps{};
  if (out == kOutRaw && (g.st_row != 1 || g.st_col % 4 != 0 || reinterpret_cast<uintptr_t>(g.state_in) % 16 != 0)) return false;
  if (g.cols > 128 || g.rows % 8 != 0 || g.seglen % kQ != 0 || reinterpret_cast<uintptr_t>(g.out) % 16 != 0 ||
      !make_map(maps.k, g.k, g.cols, g, batch, kHalf) || !make_map(maps.r, g.r, g.rows, g, batch, kHalf) ||
      (out != kOutNone && !make_map(maps.q, g.q, g.cols, g, batch, kHalf)))
    return false;
  auto go = [&](auto cols) {
    constexpr int C = decltype(cols)::value;
    if (!rev && out == kOutNone) launch<T, C, 64, false, kOutNone, true>(g, maps, batch, st);
    else if (!rev && out == kOutY) launch<T, C, 64, false, kOutY, true>(g, maps, batch, st);
    else if (rev && out == kOutNone) launch<T, C, 64, true, kOutNone, true>(g, maps, batch, st);
    else if (rev && out == kOutDx) launch<T, C, 64, true, kOutDx, false>(g, maps, batch, st);
    else if (out == kOutRaw && g.rows <= 64) {
      if (rev) launch<T, C, 64, true, kOutRaw, false>(g, maps, batch, st);
      else launch<T, C, 64, false, kOutRaw, false>(g, maps, batch, st);
    } else if (out == kOutRaw) {
      if (rev) launch<T, C, 128, true, kOutRaw, false>(g, maps, batch, st);
      else launch<T, C, 128, false, kOutRaw, false>(g, maps, batch, st);
    } else require(false, "unknown walk", FHE_ERR_INTERNAL);
  };
  // without a carried state a segment is one chunk
  require(out == kOutNone || out == kOutY || g.seglen == kQ, "segment of more than one chunk", FHE_ERR_INTERNAL);
  if (g.cols <= 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
  return true;
}

template bool launch_scan_tc<__nv_bfloat16>(RecArgs, bool, int, uint32_t, cudaStream_t);
template bool launch_scan_tc<__half>(RecArgs, bool, int, uint32_t, cudaStream_t);

uint64_t scan_tc_timeouts() {
  uint64_t sum = 0;
  for (uint64_t left = g_used_devices.load(std::memory_order_relaxed); left; left &= left - 1) {
    DeviceGuard dev(__builtin_ctzll(left));
    unsigned v = 0;
    FHE_CUDA(cudaMemcpyFromSymbol(&v, g_scan_timeouts, sizeof(v)));
    sum += v;
  }
  return sum;
}

void set_scan_wait_limit(uint32_t polls) { g_wait_limit.store(polls, std::memory_order_relaxed); }

}  // namespace fhe
