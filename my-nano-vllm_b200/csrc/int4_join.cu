// Joins the parts of row groups that the 4-bit attention kernels' even cuts left in several CTAs.
//
// Part c has the output o_c of its own positions, and their sum l_c for the reference maximum m_c; with M = max m_c
//   out = sum_c w_c o_c,  w_c = 2^(m_c - M) l_c / sum_d 2^(m_d - M) l_d,
// added in the order of the parts.  Means weighted by 0 .. 1 stay inside fp32 wherever the values do; sums of p v
// times a part's l would not.  2^(m_c - M) is put in as its root, twice: it may be below fp32's range where its product with
// large values is not.  CTA i takes what the cut of CTA i says.  Bound by latency (descriptor, maxima, sums,
// output: three dependent accesses of L2), so few rows with many parts are shared by up to four CTAs and their warps,
// with eight parts of a warp in flight, and many rows with few parts go four to a warp (4 rows of 55 parts: 2 us; one
// CTA for a pair, maxima first: 6).
#include "int4_attention.cuh"

namespace fp8attn {
namespace {

constexpr int kWarps = 8;
constexpr int kFewBlocks = 4;  // CTAs that share the rows of a cut
constexpr int kAtOnce = 8;  // parts of which a warp has the loads in flight

// y += x w root.
__device__ __forceinline__ void add_part(float4& y, const float4& x, float w, float root) {
  y.x = fmaf(x.x * root, w, y.x);
  y.y = fmaf(x.y * root, w, y.y);
  y.z = fmaf(x.z * root, w, y.z);
  y.w = fmaf(x.w * root, w, y.w);
}
__device__ __forceinline__ float root_of(float m, float top) { return ex2(0.5f * (m - top)); }  // of 2^(m - top)

__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : __fdiv_rn(1.f, sum); }

__device__ __forceinline__ void store_row(const Int4AttnParams& p, const Cut& cut, int row, int lane, const float4& y) {
  const int r = cut.first_row + row, token = r / p.group;
  const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
  *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(cut.token) + token) * p.out_row_stride +
                            (cut.head + r - token * p.group) * kHeadDim + 4 * lane) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// At most 32 rows, up to as many parts as there are CTAs: several warps of a row take parts in turn, and their sums are
// added in order.
__device__ __forceinline__ void join_few(const Int4AttnParams& p, const Int4JoinList& list, int index, int block) {
  __shared__ float4 sum_o[kWarps][32];
  __shared__ float2 sum_ml[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cut cut = reinterpret_cast<const Cut*>(list.cuts)[index];
  const int parts = cut.parts, part_size = list.rows * (kHeadDim + 2);
  if (parts == 0) return;
  const float* first = list.partials + static_cast<int64_t>(cut.slot) * part_size;
  const float* later = list.partials + static_cast<int64_t>(2 * index) * part_size;
  auto part = [&](int j) { return j == 0 ? first : later + static_cast<int64_t>(2 * j) * part_size; };
  const int ml_at = list.rows * kHeadDim;
  const int each = (cut.rows + list.blocks - 1) / list.blocks, begin = block * each, end = min(begin + each, cut.rows);
  if (begin >= end) return;
  const int share = max(1, min(kWarps / (end - begin), parts));  // warps of a row
  const int at_once = kWarps / share;                            // rows
  for (int row0 = begin; row0 < end; row0 += at_once) {
    const int row = row0 + warp / share, turn = warp % share;
    const bool mine = warp < at_once * share && row < end;
    float mx = kNone, sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = turn; mine && j0 < parts; j0 += kAtOnce * share) {
      float2 ml[kAtOnce];
      float4 x[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int j = j0 + i * share;
        ml[i] = make_float2(kNone, 0.f);
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j < parts) {
          ml[i] = *reinterpret_cast<const float2*>(part(j) + ml_at + 2 * row);
          x[i] = *reinterpret_cast<const float4*>(part(j) + row * kHeadDim + 4 * lane);
        }
      }
      const float was = mx;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) mx = fmaxf(mx, ml[i].x);
      const float old_root = root_of(was, mx), before = sum * old_root;
      sum = before * old_root;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        ml[i].x = root_of(ml[i].x, mx);
        ml[i].y *= ml[i].x;
        sum = fmaf(ml[i].y, ml[i].x, sum);
      }
      const float inv = inverse(sum);
      const float4 old = y;
      y = make_float4(0.f, 0.f, 0.f, 0.f);
      add_part(y, old, before * inv, old_root);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) add_part(y, x[i], ml[i].y * inv, ml[i].x);
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
        for (int w = 0; w < share; ++w) sum = fmaf(sum_ml[warp + w].y, ex2(sum_ml[warp + w].x - top), sum);
        const float inv = inverse(sum);
        for (int w = 0; w < share; ++w) {
          const float root = root_of(sum_ml[warp + w].x, top);
          add_part(y, sum_o[warp + w][lane], sum_ml[warp + w].y * root * inv, root);
        }
      }
    }
    if (mine && turn == 0) store_row(p, cut, row, lane, y);
  }
}

// Up to kInt4LongRows rows, four to a warp.
constexpr int kRowsPerCta = 4 * kWarps;
__device__ __forceinline__ void join_many(const Int4AttnParams& p, const Int4JoinList& list, int index, int block) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cut cut = reinterpret_cast<const Cut*>(list.cuts)[index];
  const int parts = cut.parts, part_size = list.rows * (kHeadDim + 2), row0 = block * kRowsPerCta + 4 * warp;
  if (parts == 0 || row0 >= cut.rows) return;
  const float* first = list.partials + static_cast<int64_t>(cut.slot) * part_size;
  const float* later = list.partials + static_cast<int64_t>(2 * index) * part_size;
  auto part = [&](int j) { return j == 0 ? first : later + static_cast<int64_t>(2 * j) * part_size; };
  const int ml_at = list.rows * kHeadDim + 2 * row0;
  float mx[4] = {kNone, kNone, kNone, kNone}, inv[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = lane; j < parts; j += 32) {
    const float4 a = *reinterpret_cast<const float4*>(part(j) + ml_at);  // (m, l) of two rows
    const float4 b = *reinterpret_cast<const float4*>(part(j) + ml_at + 4);
    mx[0] = fmaxf(mx[0], a.x);
    mx[1] = fmaxf(mx[1], a.z);
    mx[2] = fmaxf(mx[2], b.x);
    mx[3] = fmaxf(mx[3], b.z);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], off));
  for (int j = lane; j < parts; j += 32) {
    const float4 a = *reinterpret_cast<const float4*>(part(j) + ml_at);
    const float4 b = *reinterpret_cast<const float4*>(part(j) + ml_at + 4);
    inv[0] = fmaf(a.y, ex2(a.x - mx[0]), inv[0]);
    inv[1] = fmaf(a.w, ex2(a.z - mx[1]), inv[1]);
    inv[2] = fmaf(b.y, ex2(b.x - mx[2]), inv[2]);
    inv[3] = fmaf(b.w, ex2(b.z - mx[3]), inv[3]);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < 4; ++k) inv[k] += __shfl_xor_sync(0xffffffffu, inv[k], off);
#pragma unroll
  for (int k = 0; k < 4; ++k) inv[k] = inverse(inv[k]);
  float4 y[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (int j = 0; j < parts; ++j) {
    const float4 a = *reinterpret_cast<const float4*>(part(j) + ml_at);
    const float4 b = *reinterpret_cast<const float4*>(part(j) + ml_at + 4);
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const float4*>(part(j) + (row0 + k) * kHeadDim + 4 * lane);
    const float r0 = root_of(a.x, mx[0]);
    add_part(y[0], x[0], a.y * r0 * inv[0], r0);
    const float r1 = root_of(a.z, mx[1]);
    add_part(y[1], x[1], a.w * r1 * inv[1], r1);
    const float r2 = root_of(b.x, mx[2]);
    add_part(y[2], x[2], b.y * r2 * inv[2], r2);
    const float r3 = root_of(b.z, mx[3]);
    add_part(y[3], x[3], b.w * r3 * inv[3], r3);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (row0 + k < cut.rows) store_row(p, cut, row0 + k, lane, y[k]);
}

// CTAs [0, few.ctas * few.blocks) join the cuts of the kernel for few rows, the others those of the kernel for long
// chunks.
__global__ void __launch_bounds__(kWarps * 32, 4)
    int4_join_kernel(const __grid_constant__ Int4AttnParams p, const Int4JoinList few, const Int4JoinList many) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int at = static_cast<int>(blockIdx.x) - few.ctas * few.blocks;
  if (at < 0) {
    join_few(p, few, blockIdx.x / few.blocks, blockIdx.x % few.blocks);
  } else {
    constexpr int kBlocks = kInt4LongRows / kRowsPerCta;
    join_many(p, many, at / kBlocks, at % kBlocks);
  }
}

}  // namespace

cudaError_t launch_int4_join(const Int4AttnParams& p, Int4JoinList few, Int4JoinList many, cudaStream_t stream) {
  // the last CTA's range ends with a pair
  few.ctas = few.ctas > 1 ? few.ctas - 1 : 0;
  many.ctas = many.ctas > 1 ? many.ctas - 1 : 0;
  few.blocks = few.rows < kFewBlocks ? few.rows : kFewBlocks;
  const int blocks = few.ctas * few.blocks + many.ctas * (kInt4LongRows / kRowsPerCta);
  if (blocks == 0) return cudaSuccess;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, int4_join_kernel, p, few, many);
}

}  // namespace fp8attn
