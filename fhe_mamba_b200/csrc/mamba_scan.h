// What the two forms of the state recurrence share: its arguments.
#pragma once
#include "mamba_ops.h"

namespace fhe {

struct Src {
  const void* p;
  int64_t sb, sl, sh;  // batch, token, head (or group)
  uint32_t share;      // heads per index of the head axis
  template <class T>
  __device__ const T* at(uint32_t b, uint32_t h) const {
    return static_cast<const T*>(p) + (int64_t)b * sb + (int64_t)(h / share) * sh;
  }
};

struct Gate {
  const float* p;
  int64_t sb, sl, sh;
};

struct RecArgs {
  Src r, k, q;
  Gate write, log_decay;  // write.p == nullptr: 1
  const int32_t* lengths;
  uint32_t length, heads, rows, cols, seglen, nseg;
  const float* d;         // OUT 1, 2
  Gate out_scale;         // OUT 2: o is scaled by it
  const float* state_in;  // slot base, or nullptr for zeros
  float* state_out;       // or nullptr
  // element (b, h, segment, row, col) of the states
  int64_t in_bh, in_seg, out_bh, out_seg, st_row, st_col;
  float* seg_decay;  // STATE pass: product of the segment's decays [bh][nseg]
  void* out;
  bool vec;  // r, k and q may be read four elements at a time
  int* bad;            // set by the tensor-core form when a product of an output is not finite
  uint32_t wait_limit;  // polls of the tensor-core form's waits
  const int* only_if;  // the fp32 walk does nothing while it is 0 (nullptr: always runs)
};

enum { kOutNone = 0, kOutY = 1, kOutDx = 2, kOutRaw = 3 };

// The tensor-core form (mamba_scan_tc.cu) for bfloat16 and float16; false, with
// nothing launched, for sizes and layouts that it does not take.
template <class T>
bool launch_scan_tc(RecArgs g, bool rev, int out, uint32_t batch, cudaStream_t st);
uint64_t scan_tc_timeouts();  // over all devices
void set_scan_wait_limit(uint32_t polls);

}  // namespace fhe
