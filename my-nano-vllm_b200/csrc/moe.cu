// A mixture-of-experts layer for a few tokens, in the FP8 block-scaled format of fp8linear.cu.
//
//   l = x Wr^T;  p = softmax(l);  S = the top_k largest p (ties: the lower expert first);
//   c = p_S, divided by its sum if renormalised;
//   for each e of S:  g, u = the halves of xq . w13[e]^T;  h = g / (1 + exp(-g)) u;
//                     hq, d = h quantised per 128 columns (a = max|h|, d = a / 448 or 1);
//                     y_e = hq . w2[e]^T;
//   out = bf16(sum over S, in order, of c_e y_e)
//
// Products are block scaled: the exact dot of 128 columns times (activation scale * weight scale),
// summed over the blocks in fp32.  A slot is a (token, place in its top-k) pair, n = T top_k of them.
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace fp8attn {
namespace {

constexpr int kBlk = 128;

__device__ __forceinline__ float bf16_to_f32(uint16_t b) {
  return __uint_as_float(static_cast<uint32_t>(b) << 16);
}
__device__ __forceinline__ float e4m3_to_f32(uint8_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

// ------------------------------------------------------------------ router
// One CTA per token.  Logits: fp32 products of 8 columns at a time, added up in fp64, so that which
// experts are chosen does not hang on the order of a sum.
constexpr int kRouterThreads = 256;
constexpr int kExpertsPerLane = kMoeMaxExperts / 32;

__global__ void __launch_bounds__(kRouterThreads) moe_router_kernel(const MoeParams p) {
  __shared__ float logits[kMoeMaxExperts];
  const int64_t token = blockIdx.x;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint16_t* x = p.x + token * p.x_row_stride;
  for (int e = warp; e < p.E; e += kRouterThreads / 32) {
    const uint16_t* w = p.router + static_cast<int64_t>(e) * p.H;
    double acc = 0.0;
    for (int c = 8 * lane; c < p.H; c += 256) {
      float s = 0.f;
      for (int i = 0; i < 8; ++i) s = fmaf(bf16_to_f32(x[c + i]), bf16_to_f32(w[c + i]), s);
      acc += s;
    }
    for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if (lane == 0) logits[e] = static_cast<float>(acc);
  }
  __syncthreads();
  if (warp != 0) return;
  // top-k: every lane keeps experts lane, lane + 32, ...; a NaN logit is chosen last
  float v[kExpertsPerLane];
  uint32_t taken = 0;
#pragma unroll
  for (int j = 0; j < kExpertsPerLane; ++j) {
    const int e = lane + 32 * j;
    v[j] = e < p.E ? logits[e] : 0.f;
    if (e >= p.E) taken |= 1u << j;
  }
  float top = 0.f, chosen = 0.f;
  int my_id = 0;
  for (int k = 0; k < p.top_k; ++k) {
    float best = -INFINITY;
    int at = INT_MAX;
#pragma unroll
    for (int j = 0; j < kExpertsPerLane; ++j) {
      const float c = v[j] == v[j] ? v[j] : -INFINITY;
      if (!((taken >> j) & 1u) && (at == INT_MAX || c > best)) {
        best = c;
        at = lane + 32 * j;
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const float ob = __shfl_xor_sync(0xffffffffu, best, off);
      const int oa = __shfl_xor_sync(0xffffffffu, at, off);
      if (oa != INT_MAX && (at == INT_MAX || ob > best || (ob == best && oa < at))) {
        best = ob;
        at = oa;
      }
    }
    if (k == 0) top = best;
    if ((at & 31) == lane) taken |= 1u << (at >> 5);
    if (lane == k) {
      my_id = at;
      chosen = logits[at];
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < kExpertsPerLane; ++j)
    if (lane + 32 * j < p.E) sum += expf(v[j] - top);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  float c = lane < p.top_k ? expf(chosen - top) / sum : 0.f;
  if (p.renormalize) {
    float total = c;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    c /= total;
  }
  if (lane < p.top_k) {
    p.ids[token * p.top_k + lane] = my_id;
    p.weights[token * p.top_k + lane] = c;
  }
}

// ------------------------------------------------------------------ products
// Sum over the blocks of one weight row, the activation row (values and scales) in shared memory.
__device__ float block_scaled_dot(const uint8_t* w, const uint16_t* w_scale, const float* a,
                                  const float* a_scale, int K) {
  float acc = 0.f;
  for (int kb = 0; kb < K / kBlk; ++kb) {
    float d = 0.f;
    for (int c = 0; c < kBlk; ++c) d = fmaf(a[kb * kBlk + c], e4m3_to_f32(w[kb * kBlk + c]), d);
    acc = fmaf(d, a_scale[kb] * bf16_to_f32(w_scale[kb]), acc);
  }
  return acc;
}

// CTA (slot, 128 columns of I): threads 0-127 the gate rows, 128-255 the up rows.
__global__ void __launch_bounds__(256) moe_gate_up_kernel(const MoeParams p) {
  extern __shared__ float sh[];
  __shared__ float up[kBlk], warp_max[4];
  const int slot = blockIdx.x, ib = blockIdx.y, t = threadIdx.x;
  const int64_t token = slot / p.top_k;
  const int e = p.ids[slot];
  const int kc = p.H / kBlk;
  float *a = sh, *as = sh + p.H;
  for (int c = t; c < p.H; c += 256) a[c] = e4m3_to_f32(p.xq[token * p.xq_row_stride + c]);
  for (int c = t; c < kc; c += 256) as[c] = bf16_to_f32(p.x_scale[token * kc + c]);
  __syncthreads();
  const int r = t & 127, half = t >> 7;
  const int64_t row = static_cast<int64_t>(e) * 2 * p.I + half * p.I + ib * kBlk + r;
  const float y = block_scaled_dot(p.w13 + row * p.H, p.w13_scale + row / kBlk * kc, a, as, p.H);
  if (half) up[r] = y;
  __syncthreads();
  float h = 0.f;
  if (!half) {
    h = __fdiv_rn(y, 1.0f + expf(-y)) * up[r];
    float m = fmaxf(fabsf(h), 0.f);
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if ((r & 31) == 0) warp_max[r / 32] = m;
  }
  __syncthreads();
  if (half) return;
  const float m = fmaxf(fmaxf(warp_max[0], warp_max[1]), fmaxf(warp_max[2], warp_max[3]));
  float scale = __fdiv_rn(m, 448.0f);
  if (!(scale > 0.f)) scale = 1.0f;
  p.hq[static_cast<int64_t>(slot) * p.I + ib * kBlk + r] =
      static_cast<uint8_t>(f32x2_to_e4m3x2(__fdiv_rn(h, scale), 0.f) & 0xFFu);
  if (r == 0)
    p.h_scale[static_cast<int64_t>(slot) * (p.I / kBlk) + ib] =
        __bfloat16_as_ushort(__float2bfloat16_rn(scale));
}

// CTA (slot, 128 columns of H).
__global__ void __launch_bounds__(128) moe_down_kernel(const MoeParams p) {
  extern __shared__ float sh[];
  const int slot = blockIdx.x, hb = blockIdx.y, t = threadIdx.x;
  const int e = p.ids[slot];
  const int kc = p.I / kBlk;
  float *a = sh, *as = sh + p.I;
  for (int c = t; c < p.I; c += 128) a[c] = e4m3_to_f32(p.hq[static_cast<int64_t>(slot) * p.I + c]);
  for (int c = t; c < kc; c += 128) as[c] = bf16_to_f32(p.h_scale[static_cast<int64_t>(slot) * kc + c]);
  __syncthreads();
  const int64_t row = static_cast<int64_t>(e) * p.H + hb * kBlk + t;
  p.y[static_cast<int64_t>(slot) * p.H + hb * kBlk + t] =
      block_scaled_dot(p.w2 + row * p.I, p.w2_scale + row / kBlk * kc, a, as, p.I);
}

__global__ void __launch_bounds__(128) moe_combine_kernel(const MoeParams p) {
  const int64_t token = blockIdx.x;
  const int c = blockIdx.y * 128 + threadIdx.x;
  float acc = 0.f;
  for (int k = 0; k < p.top_k; ++k) {
    const int64_t slot = token * p.top_k + k;
    acc = fmaf(p.weights[slot], p.y[slot * p.H + c], acc);
  }
  p.out[token * p.out_row_stride + c] = __bfloat16_as_ushort(__float2bfloat16_rn(acc));
}

}  // namespace

int64_t moe_layout(MoeParams& p, void* workspace, int num_sms) {
  (void)num_sms;
  uint8_t* const base = static_cast<uint8_t*>(workspace);
  int64_t off = 0;
  auto take = [&](auto*& ptr, int64_t bytes) {
    if (base != nullptr && ptr == nullptr)
      ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(base + off);
    off += (bytes + 255) / 256 * 256;
  };
  const int64_t n = p.T * p.top_k;
  take(p.ids, n * 4);      // where the caller gives none
  take(p.weights, n * 4);
  take(p.hq, n * p.I);
  take(p.h_scale, n * (p.I / kBlk) * 2);
  take(p.y, n * p.H * 4);
  return off;
}

cudaError_t launch_moe(const MoeParams& p, int num_sms, cudaStream_t stream) {
  (void)num_sms;
  const unsigned n = static_cast<unsigned>(p.T * p.top_k);
  moe_router_kernel<<<static_cast<unsigned>(p.T), kRouterThreads, 0, stream>>>(p);
  const size_t sh1 = (p.H + p.H / kBlk) * 4, sh2 = (p.I + p.I / kBlk) * 4;
  if (sh1 > 200 * 1024 || sh2 > 200 * 1024) return cudaErrorInvalidValue;
  cudaFuncSetAttribute(moe_gate_up_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  cudaFuncSetAttribute(moe_down_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  moe_gate_up_kernel<<<dim3(n, p.I / kBlk), 256, sh1, stream>>>(p);
  moe_down_kernel<<<dim3(n, p.H / kBlk), 128, sh2, stream>>>(p);
  moe_combine_kernel<<<dim3(static_cast<unsigned>(p.T), p.H / kBlk), 128, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fp8attn
