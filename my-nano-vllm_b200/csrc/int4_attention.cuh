// What the two kernels of attention over the 4-bit cache share (int4_decode.cu: few query rows of a kv head,
// int4_prefill.cu: many): the work is units of 128 positions in an order, cut into equal ranges, one for each CTA,
// wherever the cuts fall; the parts of a pair (row group, kv head) that was cut are joined by a kernel of its own.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace fp8attn {
namespace {

constexpr float kNone = -3.402823466e38f;

// mbar_wait with its polling loop out of line, for a whole warp.
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, int* err) { return mbar_wait(bar, parity, err); }
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity) || wait_long(bar, parity, err));
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

// First unit of CTA i of n over u units, and the CTA that has unit x.
__device__ __forceinline__ int64_t range_begin(int64_t i, int64_t n, int64_t u) { return i * u / n; }
__device__ __forceinline__ int64_t owner(int64_t x, int64_t n, int64_t u) { return ((x + 1) * n - 1) / u; }

}  // namespace
}  // namespace fp8attn
