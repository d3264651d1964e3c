// A paged key/value cache of 4-bit codes: rows quantised as they are written, and read back.
//
// A row is one token of one kv head, 128 values x:
//   low = min x,  step = bf16((max x - min x) / 15),
//   code = the integer nearest to (x - low) / step (ties to even) in 0..15 (0 where step is 0),
//   and the row stands for low + step * code.
// low is one of the row's own bf16 values and so exact.  Codes are taken with the rounded step, so
// that its rounding (2^-9) costs the largest value at most 15 * 2^-9 = 0.03 of a step.  A row with a
// NaN or an infinity, or whose range passes bf16's, has a NaN as its step and reads as NaN.
//
// Layout: codes [num_blocks, KVH, block_size, 64] bytes, value 2 i in the low half of byte i and
// 2 i + 1 in the high half; (k step, k low, v step, v low) as bf16 [num_blocks, KVH, block_size, 4].  A
// page holds the rows of one head one after another, so 16 tokens of a head are 1 KB in one piece: the
// attention kernels' tiles are whole DRAM bursts although a row has only 64 bytes.
//
// Both kernels are bound by HBM (512 bytes of K and V in 16 bits and 136 in 4 for each token and
// head).  Sixteen threads share a row of K and the same row of V, 8 values each: a 16-byte access
// on the 16-bit side, a word of 8 codes on the other.  Consecutive rows of a CTA are consecutive tokens
// of one head, which share pages, so that their 64-byte rows leave as whole lines.
#include "common.cuh"
#include "kernels.h"

namespace fp8attn {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 16;  // consecutive tokens of a head that a CTA's 16 rows are

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t w) {
  return *reinterpret_cast<__nv_bfloat162*>(&w);
}
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }

struct Row {
  int64_t token;
  int head;
  int64_t cache_row;  // -1: none
};

// Thread's row: tokens in groups of 16, heads inside a group, tokens inside a head.
__device__ __forceinline__ Row row_of(const Int4RowsParams& p) {
  const uint32_t unit = blockIdx.x * (kThreads / 16) + threadIdx.x / 16;
  const uint32_t group = unit / (kTokens * p.num_kv_heads);
  const uint32_t rest = unit - group * (kTokens * p.num_kv_heads);
  Row r;
  r.head = static_cast<int>(rest / kTokens);
  r.token = static_cast<int64_t>(group) * kTokens + rest % kTokens;
  r.cache_row = -1;
  if (r.token < p.num_tokens) {
    const int slot = ldg_keep(p.slot_mapping + r.token);
    if (slot >= 0 && slot < p.num_slots) {
      const uint32_t page = static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.block_size);
      const uint32_t place = static_cast<uint32_t>(slot) - page * p.block_size;
      r.cache_row = (static_cast<int64_t>(page) * p.num_kv_heads + r.head) * p.block_size + place;
    }
  }
  return r;
}

// The code of a value whose quotient lies near the border between two codes (or of a row whose step has
// no inverse in fp32): x - low as an exact sum of two floats, compared with (k + 1/2) step, which is exact
// in fp32 (5 + 8 bits).
__device__ __noinline__ uint32_t code_exact(float x, float low, float step) {
  if (!(step > 0.f)) return 0;
  const float t = x - low;
  const float z = t - x;                            // t + rest = x - low exactly (two-sum)
  const float rest = (x - (t - z)) + (-low - z);
  const float k = floorf(fminf(__fdiv_rn(t, step), 15.f));
  const float over = (t - (k + 0.5f) * step) + rest;  // its sign is exact: t is next to the border
  const uint32_t n = static_cast<uint32_t>(k);
  const uint32_t up = over > 0.f || (over == 0.f && (n & 1u)) ? n + 1 : n;
  return up > 15 ? 15 : up;
}

// Eight values of a row (16 lanes) -> their codes; the row's step and low as two bf16 in *scale.
__device__ __forceinline__ uint32_t quantise8(uint4 raw, uint32_t* scale) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  // minimum and maximum on packed pairs; NaNs go through, infinities come out
  __nv_bfloat162 mn = __hmin2_nan(__hmin2_nan(as_bf162(w[0]), as_bf162(w[1])),
                                  __hmin2_nan(as_bf162(w[2]), as_bf162(w[3])));
  __nv_bfloat162 mx = __hmax2_nan(__hmax2_nan(as_bf162(w[0]), as_bf162(w[1])),
                                  __hmax2_nan(as_bf162(w[2]), as_bf162(w[3])));
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) {
    mn = __hmin2_nan(mn, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(mn), off)));
    mx = __hmax2_nan(mx, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(mx), off)));
  }
  const __nv_bfloat16 lowest = __hmin_nan(__low2bfloat16(mn), __high2bfloat16(mn));
  const __nv_bfloat16 highest = __hmax_nan(__low2bfloat16(mx), __high2bfloat16(mx));
  const float low = __bfloat162float(lowest);
  // no second rounding: (max - min) / 15 lies on the border between two bf16 values only if max - min is
  // exact in fp32, and then the quotient is exact too
  const __nv_bfloat16 stepb = __float2bfloat16_rn(__fdiv_rn(__bfloat162float(highest) - low, 15.0f));
  const float step = __bfloat162float(stepb);
  if (!(step < INFINITY)) {
    *scale = 0x7FFFu | static_cast<uint32_t>(__bfloat16_as_ushort(lowest)) << 16;
    return 0;
  }
  *scale = static_cast<uint32_t>(__bfloat16_as_ushort(stepb)) |
           static_cast<uint32_t>(__bfloat16_as_ushort(lowest)) << 16;
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  // quotients from the inverse are off by less than 16 * 3 * 2^-24 = 3e-6; within 2^-16 of a border the
  // exact comparison decides
  const float inv = __fdiv_rn(1.0f, step);
  const uint64_t inv2 = f2_pack(inv, inv), low2 = f2_pack(low, low);
  const uint64_t magic2 = f2_pack(12582912.f, 12582912.f);
  uint32_t code = 0;
  float worst = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t q = f2_mul(f2_sub(f2_pack(x[i], x[i + 1]), low2), inv2);
    const uint64_t m = f2_add(q, magic2);  // the nearest integer in the low mantissa bits
    const uint64_t d = f2_sub(q, f2_sub(m, magic2));
    float m0, m1, d0, d1;
    f2_unpack(m, m0, m1);
    f2_unpack(d, d0, d1);
    worst = fmaxf(worst, fmaxf(fabsf(d0), fabsf(d1)));
    // a quotient is at most 15.1: the rounding of step leaves no code above 15
    code |= (__float_as_uint(m0) & 15u) << (4 * i) | (__float_as_uint(m1) & 15u) << (4 * i + 4);
  }
  if (!(worst < 0.5f - 1.0f / 65536.0f) || !(inv < INFINITY) || !(inv > 1.0e-37f)) {
    code = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = i < 2 ? w[0] : i < 4 ? w[1] : i < 6 ? w[2] : w[3];
      code |= code_exact(__uint_as_float(i & 1 ? bits & 0xFFFF0000u : bits << 16), low, step) << (4 * i);
    }
  }
  return code;
}

template <bool kVec>
__device__ __forceinline__ uint4 load8(const uint16_t* src) {
  if constexpr (kVec) {
    return ldg_keep_v4(src);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = static_cast<uint32_t>(__ldg(src + 2 * k)) | static_cast<uint32_t>(__ldg(src + 2 * k + 1)) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool kVec>
__global__ void __launch_bounds__(kThreads) int4_store_kernel(const Int4RowsParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Row r = row_of(p);
  const int lane = threadIdx.x & 15;
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (r.token < p.num_tokens) {
    k = load8<kVec>(p.key + r.token * p.key_token_stride + r.head * p.key_head_stride + 8 * lane);
    v = load8<kVec>(p.value + r.token * p.value_token_stride + r.head * p.value_head_stride + 8 * lane);
  }
  uint32_t ks, vs;
  const uint32_t kc = quantise8(k, &ks), vc = quantise8(v, &vs);  // every lane shuffles
  if (r.cache_row < 0) return;
  reinterpret_cast<uint32_t*>(p.k_cache)[r.cache_row * 16 + lane] = kc;
  reinterpret_cast<uint32_t*>(p.v_cache)[r.cache_row * 16 + lane] = vc;
  if (lane == 0) reinterpret_cast<uint2*>(p.kv_scale)[r.cache_row] = make_uint2(ks, vs);
}

// Eight codes of a row -> low + step * code, rounded once from fp32 (the product is exact).
__device__ __forceinline__ uint4 restore8(uint32_t code, uint32_t scale) {
  const float step = __uint_as_float(scale << 16), low = __uint_as_float(scale & 0xFFFF0000u);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = fmaf(static_cast<float>(code >> (8 * i) & 15u), step, low);
    const float b = fmaf(static_cast<float>(code >> (8 * i + 4) & 15u), step, low);
    w[i] = as_u32(__floats2bfloat162_rn(a, b));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ void __launch_bounds__(kThreads) int4_load_kernel(const Int4RowsParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Row r = row_of(p);
  if (r.token >= p.num_tokens) return;
  const int lane = threadIdx.x & 15;
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (r.cache_row >= 0) {
    const uint32_t kc = reinterpret_cast<const uint32_t*>(p.k_cache)[r.cache_row * 16 + lane];
    const uint32_t vc = reinterpret_cast<const uint32_t*>(p.v_cache)[r.cache_row * 16 + lane];
    const uint2 scale = reinterpret_cast<const uint2*>(p.kv_scale)[r.cache_row];
    k = restore8(kc, scale.x);
    v = restore8(vc, scale.y);
  }
  const int64_t at = (r.token * p.num_kv_heads + r.head) * kHeadDim + 8 * lane;
  *reinterpret_cast<uint4*>(p.key_out + at) = k;
  *reinterpret_cast<uint4*>(p.value_out + at) = v;
}

template <typename Kernel>
cudaError_t launch_rows(Kernel* kernel, const Int4RowsParams& p, cudaStream_t stream) {
  const int64_t groups = (p.num_tokens + kTokens - 1) / kTokens;
  const int64_t blocks = groups * p.num_kv_heads;  // 16 rows each
  if (blocks * kTokens > UINT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_int4_store(const Int4RowsParams& p, cudaStream_t stream) {
  if (p.num_tokens == 0) return cudaSuccess;
  auto wide = [](const void* ptr, int64_t token, int64_t head) {
    return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && token % 8 == 0 && head % 8 == 0;
  };
  const bool vec = wide(p.key, p.key_token_stride, p.key_head_stride) &&
                   wide(p.value, p.value_token_stride, p.value_head_stride);
  return vec ? launch_rows(int4_store_kernel<true>, p, stream)
             : launch_rows(int4_store_kernel<false>, p, stream);
}

cudaError_t launch_int4_load(const Int4RowsParams& p, cudaStream_t stream) {
  if (p.num_tokens == 0) return cudaSuccess;
  return launch_rows(int4_load_kernel, p, stream);
}

}  // namespace fp8attn
