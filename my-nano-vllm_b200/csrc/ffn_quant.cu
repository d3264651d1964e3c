// The activations of an FP8 feed-forward block, written in 8 bits by the kernel that makes them:
//
//   add_rms_norm_quant   s = x + residual, y = s / sqrt(mean(s^2) + eps) * w,  quantised
//   silu_mul_quant       h = g / (1 + exp(-g)) * u,                           quantised
//
// Quantised as the FP8 block-scaled linear layer reads it (fp8linear.cu): per row and 128 columns
// a = max|y| (NaN left out), d = a / 448 (1 for an all-zero group), e4m3(y / d), and d as bf16.  The
// norm and the activation stay in fp32 up to that one rounding: the chain of a norm with a 16-bit
// result and a separate quantisation rounds twice and moves the row through memory once more.
//
// Bound: HBM.  A group of 128 columns is 16 lanes of 8 elements (one 16-byte load each), so its
// maximum is a 4-step shuffle and nothing but the norm's sum crosses warps.
#include "common.cuh"
#include "kernels.h"

namespace fp8attn {
namespace {

constexpr int kGroup = 128;

__device__ __forceinline__ float load_elem(uint32_t bits16, __nv_bfloat16) {
  return __uint_as_float(bits16 << 16);
}
__device__ __forceinline__ float load_elem(uint32_t bits16, __half) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits16)));
}
__device__ __forceinline__ uint32_t store_elem(float x, __nv_bfloat16) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}
__device__ __forceinline__ uint32_t store_elem(float x, __half) {
  return __half_as_ushort(__float2half_rn(x));
}

template <typename T>
__device__ __forceinline__ void widen8(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = load_elem(w[i] & 0xFFFFu, T());
    x[2 * i + 1] = load_elem(w[i] >> 16, T());
  }
}

template <typename T>
__device__ __forceinline__ uint4 narrow8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = store_elem(x[2 * i], T()) | (store_elem(x[2 * i + 1], T()) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 bytes that are read once: not kept in L1.  Not the read-only path: an output may be the
// residual itself.
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// This lane's 8 of a group's 128 values, the group being the 16 lanes of its half-warp: the e4m3
// bytes, and the group's scale.  The lanes of `mask` call together.
__device__ __forceinline__ uint2 quantise8(const float (&y)[8], float& scale, unsigned mask) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(y[i]));  // fmaxf leaves NaN out
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor_sync(mask, a, off));
  scale = __fdiv_rn(a, 448.0f);
  if (!(scale > 0.f)) scale = 1.0f;
  // y / d as y times 1 / d, an ulp from the quotient (31 instead of 60 instructions an element in the
  // SiLU kernel), but for scales whose inverse overflows
  float v[8];
  if (scale > 1.0e-37f) {
    const float inv = __frcp_rn(scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = y[i] * inv;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fdiv_rn(y[i], scale);
  }
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)  // saturating: a quotient may round to just above 448
    b[i] = f32x2_to_e4m3x2(v[2 * i], v[2 * i + 1]);
  return make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
}

__device__ __forceinline__ uint16_t bf16_bits(float x) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// ------------------------------------------------------------------ add + RMS norm + quantise
// kTpr threads per row (a power of two from 32), kVec vectors of 8 per thread: vector j of thread t
// is columns 8 (t + j kTpr).  kRows rows per CTA.
template <typename T, int kTpr, int kVec, int kRows>
__global__ void __launch_bounds__(kTpr* kRows) add_rms_norm_quant_kernel(const NormQuantParams p) {
  static_assert(kTpr % 32 == 0, "groups of 16 lanes must not straddle rows");
  constexpr int kWarps = kTpr / 32;
  __shared__ float part[kRows][kWarps];
  // launched as a programmatic dependent of the previous kernel: nothing is read before it ends
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x % kTpr, r = threadIdx.x / kTpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + r;
  const bool row_ok = row < p.M;  // whole warps; every thread reaches the barrier
  const int vecs = p.K / 8;
  uint4 xr[kVec], rr[kVec], wr[kVec];
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int v = t + j * kTpr;
    const bool ok = row_ok && v < vecs;
    xr[j] = rr[j] = wr[j] = make_uint4(0, 0, 0, 0);
    if (ok) xr[j] = load_once(p.x + row * p.x_row_stride + 8 * v);
    if (ok && p.residual != nullptr) rr[j] = load_once(p.residual + row * p.residual_row_stride + 8 * v);
    if (ok) wr[j] = __ldg(reinterpret_cast<const uint4*>(p.weight) + v);
  }
  float s[kVec][8], ss = 0.f;
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    widen8<T>(xr[j], s[j]);
    if (p.residual != nullptr) {
      float q[8];
      widen8<T>(rr[j], q);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[j][i] += q[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(s[j][i], s[j][i], ss);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  if (kWarps > 1) {
    if ((t & 31) == 0) part[r][t / 32] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) ss += part[r][w];
  }
  const float rms = rsqrtf(ss / static_cast<float>(p.K) + p.eps);
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int v = t + j * kTpr;
    const bool ok = row_ok && v < vecs;  // the 16 lanes of a group agree: vecs is a multiple of 16
    const unsigned mask = __ballot_sync(0xffffffffu, ok);
    if (!ok) continue;
    if (p.residual_out != nullptr)
      *reinterpret_cast<uint4*>(p.residual_out + row * p.K + 8 * v) = narrow8<T>(s[j]);
    float w[8], y[8];
    widen8<T>(wr[j], w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = s[j][i] * rms * w[i];
    if (p.norm_out != nullptr)
      *reinterpret_cast<uint4*>(p.norm_out + row * p.K + 8 * v) = narrow8<T>(y);
    float scale;
    const uint2 q = quantise8(y, scale, mask);
    *reinterpret_cast<uint2*>(p.q + row * p.K + 8 * v) = q;
    if ((v & 15) == 0) p.scale[row * (p.K / kGroup) + v / 16] = bf16_bits(scale);
  }
}

// ------------------------------------------------------------------ SiLU * up + quantise
constexpr int kSiluThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kSiluThreads) silu_mul_quant_kernel(const SiluQuantParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int vecs = p.I / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kSiluThreads + threadIdx.x;
  const bool ok = i < p.M * vecs;  // the 16 lanes of a group agree: vecs is a multiple of 16
  const unsigned mask = __ballot_sync(0xffffffffu, ok);
  if (!ok) return;
  const int64_t row = i / vecs;
  const int v = static_cast<int>(i - row * vecs);
  const uint16_t* src = p.gate_up + row * p.row_stride + 8 * v;
  const uint4 gr = load_once(src), ur = load_once(src + p.I);
  float g[8], u[8];
  widen8<T>(gr, g);
  widen8<T>(ur, u);
#pragma unroll
  for (int k = 0; k < 8; ++k) g[k] = __fdividef(g[k], 1.0f + expf(-g[k])) * u[k];
  float scale;
  const uint2 q = quantise8(g, scale, mask);
  *reinterpret_cast<uint2*>(p.q + row * p.I + 8 * v) = q;
  if ((v & 15) == 0) p.scale[row * (p.I / kGroup) + v / 16] = bf16_bits(scale);
}

template <typename Kernel, typename Params>
cudaError_t launch_dependent(Kernel kernel, int64_t blocks, int threads, const Params& p,
                             cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int kTpr, int kVec, int kRows>
cudaError_t launch_norm(const NormQuantParams& p, cudaStream_t stream) {
  return launch_dependent(add_rms_norm_quant_kernel<T, kTpr, kVec, kRows>, (p.M + kRows - 1) / kRows,
                          kTpr * kRows, p, stream);
}

template <typename T>
cudaError_t launch_norm_for(const NormQuantParams& p, cudaStream_t stream) {
  const int vecs = p.K / 8;
  if (vecs <= 64) return launch_norm<T, 32, 2, 4>(p, stream);
  if (vecs <= 256) return launch_norm<T, 128, 2, 2>(p, stream);
  if (vecs <= 512) return launch_norm<T, 256, 2, 1>(p, stream);
  if (vecs <= 1024) return launch_norm<T, 512, 2, 1>(p, stream);
  return launch_norm<T, 512, 4, 1>(p, stream);
}

}  // namespace

cudaError_t launch_add_rms_norm_quant(const NormQuantParams& p, cudaStream_t stream) {
  if (p.M == 0) return cudaSuccess;
  return p.fp16 ? launch_norm_for<__half>(p, stream) : launch_norm_for<__nv_bfloat16>(p, stream);
}

cudaError_t launch_silu_mul_quant(const SiluQuantParams& p, cudaStream_t stream) {
  if (p.M == 0) return cudaSuccess;
  const int64_t blocks = (p.M * (p.I / 8) + kSiluThreads - 1) / kSiluThreads;
  return p.fp16 ? launch_dependent(silu_mul_quant_kernel<__half>, blocks, kSiluThreads, p, stream)
                : launch_dependent(silu_mul_quant_kernel<__nv_bfloat16>, blocks, kSiluThreads, p,
                                   stream);
}

}  // namespace fp8attn
