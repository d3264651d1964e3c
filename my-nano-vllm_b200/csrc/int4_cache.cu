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
// Both kernels are bound by HBM (512 bytes of K and V in 16 bits and 136 in 4 for each token and head), the first
// nearly as much by instruction issue.  Eight threads share a row of K and the same row of V; thread i has values
// 8 i .. 8 i + 7 of either half, so that every access is a whole line: 16 bytes on the 16-bit side, a word of codes.  A
// CTA's rows are consecutive tokens of one head, which share pages, so that their 64-byte rows leave as whole lines.
// 8,192 tokens of 8 heads written and read back: 20.7 us (a thread for each half row, a division for each value: 39).
#include "common.cuh"
#include "kernels.h"

namespace fp8attn {
namespace {

constexpr int kThreads = 128;
constexpr int kLanes = 8;                    // threads of a row
constexpr int kTokens = kThreads / kLanes;   // consecutive tokens of a head that a CTA has

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t w) {
  return *reinterpret_cast<__nv_bfloat162*>(&w);
}
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }

// The cache row of a slot, -1 for none.  slot / block_size by a multiplication (block_inverse = 2^(31 + block_shift) /
// block_size, rounded up; exact for slots below 2^31).
__device__ __forceinline__ int64_t row_of(const Int4RowsParams& p, int slot, int head) {
  if (slot < 0 || slot >= p.num_slots) return -1;
  const uint32_t page = __umulhi(static_cast<uint32_t>(slot), p.block_inverse) >> (p.block_shift - 1);
  return (static_cast<int64_t>(page) * p.num_kv_heads + head) * p.block_size +
         (slot - static_cast<int>(page) * p.block_size);
}

// Step and lowest value of a row; the inverse that quotients are taken with first.
struct RowScale {
  float step, low, inverse;
  uint32_t packed;  // as stored
  bool plain;       // neither NaN nor at the ends of fp32's range: quotients from the inverse will do
};

__device__ __forceinline__ RowScale row_scale(__nv_bfloat16 lowest, __nv_bfloat16 highest) {
  RowScale r;
  r.low = __bfloat162float(lowest);
  const float range = __bfloat162float(highest) - r.low;
  // range / 15 rounded to nearest: a product with the rounded 1 / 15 and one correction by the exact remainder (Markstein),
  // where that stays inside fp32's normal numbers.  No second rounding: range / 15 lies on the border between
  // two bf16 values only if the range is exact in fp32, and then the quotient is exact too.
  const float k = 1.0f / 15.0f, q = range * k;
  float step = fmaf(fmaf(-15.0f, q, range), k, q);
  r.plain = range > 1.0e-30f && range < 1.0e38f;
  if (!r.plain) step = __fdiv_rn(range, 15.0f);
  const __nv_bfloat16 rounded = __float2bfloat16_rn(step);
  r.step = __bfloat162float(rounded);
  if (!(r.step < INFINITY)) r.step = __uint_as_float(0x7FFF0000u);
  r.packed = __float_as_uint(r.step) >> 16 | static_cast<uint32_t>(__bfloat16_as_ushort(lowest)) << 16;
  const float near = rcp(r.step);
  r.inverse = fmaf(fmaf(-r.step, near, 1.0f), near, near);
  return r;
}

// The code of x from a nearest integer that may be one off where the quotient lies next to a border between codes: x - low
// as an exact sum of two floats (two-sum), and its distance from code * step compared with half a step, all exact in
// fp32 next to a border (code * step has 4 + 8 bits).
__device__ __forceinline__ uint32_t settle(float x, float low, float step, int code) {
  const float t = x - low, z = t - x;
  const float rest = (x - (t - z)) + (-low - z);
  const float away = fmaf(-static_cast<float>(code), step, t), half = 0.5f * step;
  const bool above = away > 0.f;
  const float over = above ? (away - half) + rest : (-away - half) - rest;
  if (over > 0.f || (over == 0.f && (code & 1))) code += above ? 1 : -1;
  return static_cast<uint32_t>(min(max(code, 0), 15));
}

// Eight values of a row -> their codes.
__device__ __forceinline__ uint32_t quantise8(uint4 raw, const RowScale& r) {
  if (r.plain) {
    // pairs (0, 4), (1, 5), (2, 6), (3, 7): codes are gathered as numbers, 16 bits in each half of the pair
    const uint64_t low2 = f2_pack(r.low, r.low), inv2 = f2_pack(r.inverse, r.inverse);
    const uint64_t magic2 = f2_pack(12582912.f, 12582912.f), sixteen2 = f2_pack(16.f, 16.f);
    const uint64_t x[4] = {f2_pack(__uint_as_float(raw.x << 16), __uint_as_float(raw.z << 16)),
                           f2_pack(__uint_as_float(raw.x & 0xFFFF0000u), __uint_as_float(raw.z & 0xFFFF0000u)),
                           f2_pack(__uint_as_float(raw.y << 16), __uint_as_float(raw.w << 16)),
                           f2_pack(__uint_as_float(raw.y & 0xFFFF0000u), __uint_as_float(raw.w & 0xFFFF0000u))};
    float far[8], worst = 0.f;
    uint64_t sum = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      const uint64_t q = f2_mul(f2_sub(x[i], low2), inv2);
      const uint64_t k = f2_sub(f2_add(q, magic2), magic2);  // nearest integer
      f2_unpack(f2_sub(q, k), far[i], far[i + 4]);
      worst = fmaxf(worst, fmaxf(fabsf(far[i]), fabsf(far[i + 4])));
      sum = i == 3 ? k : f2_fma(sum, sixteen2, k);
    }
    float s0, s1;
    f2_unpack(f2_add(sum, f2_pack(8388608.f, 8388608.f)), s0, s1);
    uint32_t code = __byte_perm(__float_as_uint(s0), __float_as_uint(s1), 0x5410);
    // quotients are off by less than 16 * 3 * 2^-24; bf16 values fall on borders often (one value in some 300)
    constexpr float kNear = 0.5f - 1.0f / 65536.0f;
    if (worst >= kNear) {
      uint32_t near = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) near |= (fabsf(far[i]) >= kNear ? 1u : 0u) << i;
#pragma unroll 1
      while (near != 0) {
        const int i = __ffs(near) - 1;
        near &= near - 1;
        const uint32_t pair = i < 4 ? (i < 2 ? raw.x : raw.y) : (i < 6 ? raw.z : raw.w);
        const float v = __uint_as_float(i & 1 ? pair & 0xFFFF0000u : pair << 16);
        const uint32_t c = settle(v, r.low, r.step, static_cast<int>(code >> (4 * i) & 15u));
        code = (code & ~(15u << (4 * i))) | c << (4 * i);
      }
    }
    return code;
  }
  uint32_t code = 0;
  if (r.step > 0.f) {  // not NaN
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint32_t pair = i < 4 ? (i < 2 ? raw.x : raw.y) : (i < 6 ? raw.z : raw.w);
      const float v = __uint_as_float(i & 1 ? pair & 0xFFFF0000u : pair << 16);
      const float q = fminf(__fdiv_rn(v - r.low, r.step), 15.f);
      code |= settle(v, r.low, r.step, static_cast<int>(rintf(q))) << (4 * i);
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
  const int lane = threadIdx.x % kLanes, head = static_cast<int>(blockIdx.x) % p.num_kv_heads;
  const int64_t token = static_cast<int64_t>(blockIdx.x / p.num_kv_heads) * kTokens + threadIdx.x / kLanes;
  int slot = -1;
  uint4 k[2] = {}, v[2] = {};
  if (token < p.num_tokens) {
    slot = ldg_keep(p.slot_mapping + token);
    const uint16_t* key = p.key + token * p.key_token_stride + head * p.key_head_stride + 8 * lane;
    const uint16_t* value = p.value + token * p.value_token_stride + head * p.value_head_stride + 8 * lane;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      k[i] = load8<kVec>(key + 64 * i);
      v[i] = load8<kVec>(value + 64 * i);
    }
  }
  // minimum and maximum of K's row in the low half and of V's in the high half; NaNs go through, infinities come out
  auto least = [](uint4 w) {
    return __hmin2_nan(__hmin2_nan(as_bf162(w.x), as_bf162(w.y)), __hmin2_nan(as_bf162(w.z), as_bf162(w.w)));
  };
  auto most = [](uint4 w) {
    return __hmax2_nan(__hmax2_nan(as_bf162(w.x), as_bf162(w.y)), __hmax2_nan(as_bf162(w.z), as_bf162(w.w)));
  };
  const __nv_bfloat162 kmn = __hmin2_nan(least(k[0]), least(k[1])), vmn = __hmin2_nan(least(v[0]), least(v[1]));
  const __nv_bfloat162 kmx = __hmax2_nan(most(k[0]), most(k[1])), vmx = __hmax2_nan(most(v[0]), most(v[1]));
  __nv_bfloat162 mn = __hmin2_nan(__lows2bfloat162(kmn, vmn), __highs2bfloat162(kmn, vmn));
  __nv_bfloat162 mx = __hmax2_nan(__lows2bfloat162(kmx, vmx), __highs2bfloat162(kmx, vmx));
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) {  // every lane shuffles
    mn = __hmin2_nan(mn, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(mn), off)));
    mx = __hmax2_nan(mx, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(mx), off)));
  }
  const RowScale ks = row_scale(__low2bfloat16(mn), __low2bfloat16(mx));
  const RowScale vs = row_scale(__high2bfloat16(mn), __high2bfloat16(mx));
  const uint32_t kc[2] = {quantise8(k[0], ks), quantise8(k[1], ks)};
  const uint32_t vc[2] = {quantise8(v[0], vs), quantise8(v[1], vs)};
  const int64_t row = row_of(p, slot, head);
  if (row < 0) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    reinterpret_cast<uint32_t*>(p.k_cache)[row * 16 + kLanes * i + lane] = kc[i];
    reinterpret_cast<uint32_t*>(p.v_cache)[row * 16 + kLanes * i + lane] = vc[i];
  }
  if (lane == 0) reinterpret_cast<uint2*>(p.kv_scale)[row] = make_uint2(ks.packed, vs.packed);
}

// Eight codes of a row -> low + step * code, rounded once from fp32 (the product is exact).  A code under the exponent of
// 2^23 is that much more than code * 16^i; one multiply-add takes both away.
__device__ __forceinline__ uint4 restore8(uint32_t code, uint32_t scale) {
  const float step = __uint_as_float(scale << 16), low = __uint_as_float(scale & 0xFFFF0000u);
  const uint64_t step2 = f2_pack(step, step), low2 = f2_pack(low, low);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t from = i < 2 ? code : code >> 16;
    constexpr float kBase = 8388608.f;
    const float f0 = i & 1 ? 1.f / 256.f : 1.f, f1 = i & 1 ? 1.f / 4096.f : 1.f / 16.f;
    const uint32_t m0 = i & 1 ? 0xF00u : 0xFu, m1 = i & 1 ? 0xF000u : 0xF0u;
    const uint64_t x = f2_pack(__uint_as_float((from & m0) | 0x4B000000u), __uint_as_float((from & m1) | 0x4B000000u));
    float a, b;
    f2_unpack(f2_fma(f2_fma(x, f2_pack(f0, f1), f2_pack(-kBase * f0, -kBase * f1)), step2, low2), a, b);
    w[i] = as_u32(__floats2bfloat162_rn(a, b));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ void __launch_bounds__(kThreads) int4_load_kernel(const Int4RowsParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x % kLanes, head = static_cast<int>(blockIdx.x) % p.num_kv_heads;
  const int64_t token = static_cast<int64_t>(blockIdx.x / p.num_kv_heads) * kTokens + threadIdx.x / kLanes;
  if (token >= p.num_tokens) return;
  const int64_t row = row_of(p, ldg_keep(p.slot_mapping + token), head);
  uint32_t kc[2] = {0, 0}, vc[2] = {0, 0};
  uint2 scale = make_uint2(0, 0);  // zeros
  if (row >= 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kc[i] = reinterpret_cast<const uint32_t*>(p.k_cache)[row * 16 + kLanes * i + lane];
      vc[i] = reinterpret_cast<const uint32_t*>(p.v_cache)[row * 16 + kLanes * i + lane];
    }
    scale = reinterpret_cast<const uint2*>(p.kv_scale)[row];
  }
  const int64_t at = (token * p.num_kv_heads + head) * kHeadDim + 8 * lane;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    *reinterpret_cast<uint4*>(p.key_out + at + 64 * i) = restore8(kc[i], scale.x);
    *reinterpret_cast<uint4*>(p.value_out + at + 64 * i) = restore8(vc[i], scale.y);
  }
}

template <typename Kernel>
cudaError_t launch_rows(Kernel* kernel, Int4RowsParams p, cudaStream_t stream) {
  const int64_t blocks = (p.num_tokens + kTokens - 1) / kTokens * p.num_kv_heads;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  p.block_shift = 1;
  while ((int64_t{1} << p.block_shift) < p.block_size) ++p.block_shift;
  const uint64_t one = uint64_t{1} << (31 + p.block_shift);
  p.block_inverse = static_cast<uint32_t>((one + p.block_size - 1) / p.block_size);
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
