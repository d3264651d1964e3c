// Rotary positions of q and k as an operator of its own: pairs (x_i, x_{i + R/2}) ("halves") or
// (x_2i, x_{2i+1}) ("interleaved") of the first R values of a head are turned by the angle whose cos
// and sin stand in the table's row of the token's position; the head's other values pass through.
//
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin      (fp32: a product and a fused multiply-add each)
//
// and one rounding to the input's type.  The table is the framework's (cos of R / 2 frequencies, then
// sin), so any scaling of positions or frequencies is in it already.
//
// Bound by HBM: each value is read and written once.  A thread turns 8 pairs (two 16-byte loads) of
// several heads of one token, so that the 64 bytes of cos and sin that it needs are loaded once for all
// of them; all loads are issued before the first is used.  Where strides, addresses or R do not allow
// 16-byte accesses, 2 pairs (4-byte accesses) or one pair at a time.
#include "common.cuh"
#include "kernels.h"

namespace fp8attn {
namespace {

constexpr int kRopeThreads = 128;

template <bool kFp16>
__device__ __forceinline__ float widen(uint32_t bits16) {
  if (kFp16) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits16)));
  return __uint_as_float(bits16 << 16);
}
template <bool kFp16>
__device__ __forceinline__ uint32_t narrow(float x) {
  if (kFp16) return __half_as_ushort(__float2half_rn(x));
  return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}
// Two at a time: one instruction, where one alone goes through the unit of the special functions.
template <bool kFp16>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  if (kFp16) return pack_f16x2(lo, hi);
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// kN 16-bit values at p, two to a word (kN = 1: in the low half).
template <int kN>
__device__ __forceinline__ void load_values(const uint16_t* p, uint32_t (&w)[(kN + 1) / 2]) {
  if constexpr (kN == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (kN == 2) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    w[0] = *p;
  }
}
template <int kN>
__device__ __forceinline__ void store_values(uint16_t* p, const uint32_t (&w)[(kN + 1) / 2]) {
  if constexpr (kN == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if constexpr (kN == 2) {
    *reinterpret_cast<uint32_t*>(p) = w[0];
  } else {
    *p = static_cast<uint16_t>(w[0]);
  }
}

// One thread: kPairs pairs (or 2 kPairs values that pass through) of kHeads heads of one token.
template <int kPairs, int kHeads, bool kInterleaved, bool kFp16>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  // programmatic dependent of the kernel before it: nothing is read before that ends
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int kW = (kPairs + 1) / 2;
  const uint32_t unit = blockIdx.x * kRopeThreads + threadIdx.x;  // < 2^32: the host's check
  const uint32_t per_token = static_cast<uint32_t>(p.chunks * p.head_groups);
  const uint32_t token = unit / per_token;
  if (token >= p.num_tokens) return;
  const int rest = static_cast<int>(unit - token * per_token);
  const int chunk = rest % p.chunks, h0 = rest / p.chunks * kHeads;
  const int heads = min(kHeads, p.num_heads + p.num_kv_heads - h0);
  const bool turned = chunk < p.turned_chunks;
  // the two runs of kPairs values
  int first, second;
  if (!turned) {
    first = p.rotary_dim + (chunk - p.turned_chunks) * 2 * kPairs;
    second = first + kPairs;
  } else if (kInterleaved) {
    first = chunk * 2 * kPairs;
    second = first + kPairs;
  } else {
    first = chunk * kPairs;
    second = first + p.rotary_dim / 2;
  }
  uint32_t a[kHeads][kW], b[kHeads][kW];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (i < heads) {
      const int h = h0 + i;
      const uint16_t* src =
          h < p.num_heads ? p.q + token * p.q_token_stride + h * p.q_head_stride
                          : p.k + token * p.k_token_stride + (h - p.num_heads) * p.k_head_stride;
      load_values<kPairs>(src + first, a[i]);
      load_values<kPairs>(src + second, b[i]);
    }
  }
  float c[kPairs], s[kPairs];
  if (turned) {
    int64_t pos = p.positions[token];
    pos = pos < 0 ? 0 : (pos >= p.max_position ? p.max_position - 1 : pos);  // stay in the table
    const float* row = p.cos_sin + pos * p.rotary_dim + chunk * kPairs;
    const float* sin_row = row + p.rotary_dim / 2;
    if constexpr (kPairs == 8) {
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 cv = __ldg(reinterpret_cast<const float4*>(row + j));
        const float4 sv = __ldg(reinterpret_cast<const float4*>(sin_row + j));
        c[j] = cv.x; c[j + 1] = cv.y; c[j + 2] = cv.z; c[j + 3] = cv.w;
        s[j] = sv.x; s[j + 1] = sv.y; s[j + 2] = sv.z; s[j + 3] = sv.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        c[j] = __ldg(row + j);
        s[j] = __ldg(sin_row + j);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (i >= heads) break;
    if (turned) {
      float x[2 * kPairs];  // the first run's values, then the second's
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        x[j] = widen<kFp16>(a[i][j / 2] >> (16 * (j & 1)) & 0xFFFFu);
        x[kPairs + j] = widen<kFp16>(b[i][j / 2] >> (16 * (j & 1)) & 0xFFFFu);
      }
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        float& x1 = x[kInterleaved ? 2 * j : j];
        float& x2 = x[kInterleaved ? 2 * j + 1 : kPairs + j];
        const float y1 = fmaf(x1, c[j], -__fmul_rn(x2, s[j]));
        const float y2 = fmaf(x2, c[j], __fmul_rn(x1, s[j]));
        x1 = y1;
        x2 = y2;
      }
#pragma unroll
      for (int j = 0; j < kW; ++j) {
        if (kPairs == 1) {
          a[i][0] = narrow<kFp16>(x[0]);
          b[i][0] = narrow<kFp16>(x[1]);
        } else {
          a[i][j] = narrow2<kFp16>(x[2 * j], x[2 * j + 1]);
          b[i][j] = narrow2<kFp16>(x[kPairs + 2 * j], x[kPairs + 2 * j + 1]);
        }
      }
    }
    const int h = h0 + i;
    uint16_t* dst =
        h < p.num_heads
            ? p.q_out + token * p.q_out_token_stride + h * p.q_out_head_stride
            : p.k_out + token * p.k_out_token_stride + (h - p.num_heads) * p.k_out_head_stride;
    store_values<kPairs>(dst + first, a[i]);
    store_values<kPairs>(dst + second, b[i]);
  }
}

template <int kPairs, int kHeads>
cudaError_t launch(RopeParams p, cudaStream_t stream) {
  p.turned_chunks = p.rotary_dim / 2 / kPairs;
  // in place, values that pass through stay where they are
  p.chunks = p.turned_chunks + (p.in_place ? 0 : (p.head_dim - p.rotary_dim) / (2 * kPairs));
  p.head_groups = (p.num_heads + p.num_kv_heads + kHeads - 1) / kHeads;
  const int64_t units = p.num_tokens * p.chunks * p.head_groups;
  if (units > UINT32_MAX - kRopeThreads) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((units + kRopeThreads - 1) / kRopeThreads));
  cfg.blockDim = dim3(kRopeThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (p.interleaved)
    return p.fp16 ? cudaLaunchKernelEx(&cfg, rope_kernel<kPairs, kHeads, true, true>, p)
                  : cudaLaunchKernelEx(&cfg, rope_kernel<kPairs, kHeads, true, false>, p);
  return p.fp16 ? cudaLaunchKernelEx(&cfg, rope_kernel<kPairs, kHeads, false, true>, p)
                : cudaLaunchKernelEx(&cfg, rope_kernel<kPairs, kHeads, false, false>, p);
}

}  // namespace

cudaError_t launch_rope(const RopeParams& p, cudaStream_t stream) {
  if (p.num_tokens == 0) return cudaSuccess;
  // the widest access that every row, run and pair of runs allows
  auto fits = [&](int pairs, uintptr_t bytes) {
    auto rows = [&](const void* ptr, int64_t token, int64_t head) {
      return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && token % pairs == 0 && head % pairs == 0;
    };
    return p.rotary_dim / 2 % pairs == 0 && (p.head_dim - p.rotary_dim) % (2 * pairs) == 0 &&
           rows(p.q, p.q_token_stride, p.q_head_stride) &&
           rows(p.q_out, p.q_out_token_stride, p.q_out_head_stride) &&
           (p.num_kv_heads == 0 || (rows(p.k, p.k_token_stride, p.k_head_stride) &&
                                    rows(p.k_out, p.k_out_token_stride, p.k_out_head_stride)));
  };
  // two heads a thread halve the loads of cos and sin, one head spreads a small call over more SMs (8,192 tokens of 40
  // heads: 30.2 us with two, 31.5 with four; one token: 2.3 us with one, 2.5 with two)
  const bool small = p.num_tokens * (p.num_heads + p.num_kv_heads) < 8192;
  if (fits(8, 16)) return small ? launch<8, 1>(p, stream) : launch<8, 2>(p, stream);
  // narrow accesses: more heads a thread, so that cos and sin weigh less (the same with 74 of 128 values turned: 53.0 us
  // with eight, 62.5 with four, 87 with two)
  if (fits(2, 4)) return small ? launch<2, 1>(p, stream) : launch<2, 8>(p, stream);
  return small ? launch<1, 1>(p, stream) : launch<1, 8>(p, stream);
}

}  // namespace fp8attn
