// What the two kernels of attention over the 4-bit cache share (int4_decode.cu: few query rows of a kv head,
// int4_prefill.cu: many): the work is units of 128 positions in an order, cut into equal ranges, one for each CTA,
// wherever the cuts fall; the parts of a pair (row group, kv head) that was cut are joined by a kernel of its own.
#pragma once
#include <climits>

#include "common.cuh"
#include "kernels.h"

namespace fp8attn {
namespace {

constexpr float kNone = -3.402823466e38f;

// A warp's wait, bounded by a number of polls (the hardware ends each after 7,800 cycles when nothing comes: a second in
// all).  Small, since it stands in many places: the roles' loops share the instruction cache.
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, int* err) {
  bool done = false;
#pragma unroll 1
  for (uint32_t polls = 0; polls < (1u << 18) && !done; ++polls) done = mbar_try_wait(bar, parity);
  done = __all_sync(0xffffffffu, done);
  if (!done) atomicExch(err, kDevErrWaitTimeout);
  return done;
}

// size bytes (a multiple of 16, both addresses too) from global to shared memory, counted on the mbarrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t size, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(size), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ float pow2(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
__device__ __forceinline__ int exponent(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 255u) - 127; }

// A pair that is cut for the first time at the end of a CTA's range: what joins its parts has to know.
struct Cut {
  int parts;  // 0: the CTA's range ends with a pair or with a later part of one
  int slot;   // of the first part; part j > 0 is the first piece of CTA + j
  int rows;   // of the row group
  int first_row;  // in the group's kv head: token * group + head
  int token, head;  // the sequence's first row of q, and the kv head's first query head
  int unused[2];
};
static_assert(sizeof(Cut) == kInt4CutBytes, "as in kernels.h");

// u units in n ranges of equal size, the first u % n of them one longer.
struct Ranges {
  int each, longer;
  __device__ __forceinline__ Ranges(int u, int n) : each(u / n), longer(u % n) {}
  __device__ __forceinline__ int begin(int i) const { return i * each + min(i, longer); }
  __device__ __forceinline__ int owner(int x) const {  // range of unit x
    const int split = longer * (each + 1);
    return x < split ? x / (each + 1) : longer + (x - split) / each;
  }
};

}  // namespace
}  // namespace fp8attn
