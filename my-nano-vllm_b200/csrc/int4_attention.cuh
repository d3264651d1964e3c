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

// First unit of CTA i of n over u units, and the CTA that has unit x.
__device__ __forceinline__ int64_t range_begin(int64_t i, int64_t n, int64_t u) { return i * u / n; }
__device__ __forceinline__ int64_t owner(int64_t x, int64_t n, int64_t u) { return ((x + 1) * n - 1) / u; }

// Joins the parts of cut pairs: CTA (i, k) those of the pair that the first kernel's CTA i left cut, of its rows from
// k R / gridDim.y on.  kJoinWarps warps share the rows; several warps of a row take parts in turn and add what they have in order.
constexpr int kJoinWarps = 8;
template <int R>
__global__ void __launch_bounds__(kJoinWarps * 32) int4_join_kernel(const __grid_constant__ Int4AttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float4 sum_o[kJoinWarps][32];
  __shared__ float2 sum_ml[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cut cut = reinterpret_cast<const Cut*>(p.cuts)[blockIdx.x];
  const int parts = cut.parts;
  const int begin = blockIdx.y * (R / gridDim.y), rows = min(cut.rows - begin, static_cast<int>(R / gridDim.y));
  if (parts == 0 || rows <= 0) return;
  constexpr int kPart = R * (kHeadDim + 2);
  const float* first = p.partials + static_cast<int64_t>(cut.slot) * kPart;
  const float* later = p.partials + static_cast<int64_t>(2 * blockIdx.x) * kPart;
  auto part = [&](int j) { return j == 0 ? first : later + static_cast<int64_t>(2 * j) * kPart; };
  const int share = max(1, min(kJoinWarps / rows, parts));  // warps of a row
  const int at_once = kJoinWarps / share;                       // rows
  for (int row0 = begin; row0 < begin + rows; row0 += at_once) {
    const int row = row0 + warp / share, turn = warp % share;
    const bool mine = warp < at_once * share && row < begin + rows;
    float mx = kNone, sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine) {
      for (int j = turn + lane * share; j < parts; j += 32 * share) mx = fmaxf(mx, part(j)[R * kHeadDim + 2 * row]);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
#pragma unroll 8
      for (int j = turn; j < parts; j += share) {
        const float2 ml = *reinterpret_cast<const float2*>(part(j) + R * kHeadDim + 2 * row);
        const float4 x = *reinterpret_cast<const float4*>(part(j) + row * kHeadDim + 4 * lane);
        const float f = ex2(ml.x - mx);
        y.x = fmaf(x.x, f, y.x);
        y.y = fmaf(x.y, f, y.y);
        y.z = fmaf(x.z, f, y.z);
        y.w = fmaf(x.w, f, y.w);
        sum = fmaf(ml.y, f, sum);
      }
    }
    if (share > 1) {
      __syncthreads();  // the rows before these have been read
      sum_o[warp][lane] = y;
      if (lane == 0) sum_ml[warp] = make_float2(mx, sum);
      __syncthreads();
      if (mine && turn == 0) {
        float top = kNone;
        for (int w = 0; w < share; ++w) top = fmaxf(top, sum_ml[warp + w].x);
        y = make_float4(0.f, 0.f, 0.f, 0.f);
        sum = 0.f;
        for (int w = 0; w < share; ++w) {
          const float f = ex2(sum_ml[warp + w].x - top);
          const float4 x = sum_o[warp + w][lane];
          y.x = fmaf(x.x, f, y.x);
          y.y = fmaf(x.y, f, y.y);
          y.z = fmaf(x.z, f, y.z);
          y.w = fmaf(x.w, f, y.w);
          sum = fmaf(sum_ml[warp + w].y, f, sum);
        }
      }
    }
    if (mine && turn == 0) {
      const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
      const int r = cut.first_row + row, token = r / p.group;
      __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(
          p.out + (static_cast<int64_t>(cut.token) + token) * p.out_row_stride +
          (cut.head + r - token * p.group) * kHeadDim + 4 * lane);
      dst[0] = __floats2bfloat162_rn(y.x * inv, y.y * inv);
      dst[1] = __floats2bfloat162_rn(y.z * inv, y.w * inv);
    }
  }
}

}  // namespace
}  // namespace fp8attn
