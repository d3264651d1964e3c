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

// 8 values as four fp32 pairs: the kernels are bound by instruction issue before HBM, and one packed
// operation serves two values.
struct Eight {
  uint64_t p[4];
};

__device__ __forceinline__ Eight widen8(const uint4& raw, __nv_bfloat16) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    e.p[i] = f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
  return e;
}
__device__ __forceinline__ Eight widen8(const uint4& raw, __half) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    e.p[i] = f2_pack(f.x, f.y);
  }
  return e;
}
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow2(float lo, float hi, __half) { return pack_f16x2(lo, hi); }
template <typename T>
__device__ __forceinline__ uint4 narrow8(const Eight& e) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2_unpack(e.p[i], lo, hi);
    w[i] = narrow2(lo, hi, T());
  }
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
__device__ __forceinline__ uint2 quantise8(const Eight& y, float& scale, unsigned mask) {
  float v[8], a = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f2_unpack(y.p[i], v[2 * i], v[2 * i + 1]);
    a = fmaxf(a, fmaxf(fabsf(v[2 * i]), fabsf(v[2 * i + 1])));  // fmaxf leaves NaN out
  }
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor_sync(mask, a, off));
  scale = divide_by_scale(v, a);
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
// CTA: blockDim.y rows of blockDim.x threads (whole warps), kVec vectors of 8 per thread: vector j of
// thread t is columns 8 (t + j blockDim.x).
constexpr int kNormMaxWarps = 16;

template <typename T, int kVec>
__global__ void __launch_bounds__(kNormMaxWarps * 32) add_rms_norm_quant_kernel(const NormQuantParams p) {
  __shared__ float part[kNormMaxWarps];  // a row's warps side by side
  // launched as a programmatic dependent of the previous kernel: nothing is read before it ends
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x, tpr = blockDim.x, warps = tpr / 32;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool row_ok = row < p.M;  // whole warps; every thread reaches the barrier
  const int vecs = p.K / 8;
  uint4 xr[kVec], rr[kVec], wr[kVec];
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int v = t + j * tpr;
    const bool ok = row_ok && v < vecs;
    xr[j] = rr[j] = wr[j] = make_uint4(0, 0, 0, 0);
    if (ok) xr[j] = load_once(p.x + row * p.x_row_stride + 8 * v);
    if (ok && p.residual != nullptr) rr[j] = load_once(p.residual + row * p.residual_row_stride + 8 * v);
    if (ok) wr[j] = __ldg(reinterpret_cast<const uint4*>(p.weight) + v);
  }
  Eight s[kVec];
  uint64_t sq = f2_pack(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    s[j] = widen8(xr[j], T());
    if (p.residual != nullptr) {
      const Eight q = widen8(rr[j], T());
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j].p[i] = f2_add(s[j].p[i], q.p[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sq = f2_fma(s[j].p[i], s[j].p[i], sq);
  }
  float ss, ss_hi;
  f2_unpack(sq, ss, ss_hi);
  ss += ss_hi;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  if (warps > 1) {
    float* const mine = part + threadIdx.y * warps;
    if ((t & 31) == 0) mine[t / 32] = ss;
    __syncthreads();
    ss = 0.f;
    for (int w = 0; w < warps; ++w) ss += mine[w];
  }
  const float rms = rsqrtf(ss / static_cast<float>(p.K) + p.eps);
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int v = t + j * tpr;
    const bool ok = row_ok && v < vecs;  // the 16 lanes of a group agree: vecs is a multiple of 16
    const unsigned mask = __ballot_sync(0xffffffffu, ok);
    if (!ok) continue;
    if (p.residual_out != nullptr)
      *reinterpret_cast<uint4*>(p.residual_out + row * p.K + 8 * v) = narrow8<T>(s[j]);
    const Eight w = widen8(wr[j], T());
    Eight y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y.p[i] = f2_mul(f2_mul(s[j].p[i], f2_pack(rms, rms)), w.p[i]);
    if (p.norm_out != nullptr)
      *reinterpret_cast<uint4*>(p.norm_out + row * p.K + 8 * v) = narrow8<T>(y);
    float scale;
    const uint2 q = quantise8(y, scale, mask);
    *reinterpret_cast<uint2*>(p.q + row * p.K + 8 * v) = q;
    if ((v & 15) == 0) p.scale[row * (p.K / kGroup) + v / 16] = bf16_bits(scale);
  }
}

// ------------------------------------------------------------------ SiLU * up + quantise
constexpr int kSiluThreads = 128;  // 80.2 us for 8192 x 12288, 8.5 for 333 x 25600 (256: 82.9 and 9.1)
constexpr int kSiluThreadsLog2 = 7;
static_assert(kSiluThreads == 1 << kSiluThreadsLog2, "shifts");

// A CTA (x, y) takes 256 vectors of a row from 256 y on, or, of short rows, several rows: 2^tpr_log2 threads
// a row, two vectors each (one vector a thread issued 25 instructions a value, a third of them indexing).
constexpr int kSiluVec = 2;

template <typename T>
__global__ void __launch_bounds__(kSiluThreads)
    silu_mul_quant_kernel(const SiluQuantParams p, int tpr_log2) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tpr = 1 << tpr_log2, vecs = p.I / 8;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) << (kSiluThreadsLog2 - tpr_log2)) + (threadIdx.x >> tpr_log2);
  const int v0 = blockIdx.y * (kSiluThreads * kSiluVec) + (threadIdx.x & (tpr - 1));
  const uint16_t* src = p.gate_up + row * p.row_stride + 8 * v0;
  uint4 gr[kSiluVec], ur[kSiluVec];
#pragma unroll
  for (int j = 0; j < kSiluVec; ++j) {
    const bool ok = row < p.M && v0 + j * tpr < vecs;
    gr[j] = ur[j] = make_uint4(0, 0, 0, 0);
    if (ok) {
      gr[j] = load_once(src + 8 * j * tpr);
      ur[j] = load_once(src + 8 * j * tpr + p.I);
    }
  }
  uint8_t* const q = p.q + row * p.I;
  uint16_t* const scales = p.scale + row * (p.I / kGroup);
#pragma unroll
  for (int j = 0; j < kSiluVec; ++j) {
    const int v = v0 + j * tpr;
    const bool ok = row < p.M && v < vecs;  // the 16 lanes of a group agree: vecs is a multiple of 16
    const unsigned mask = __ballot_sync(0xffffffffu, ok);
    if (!ok) continue;
    Eight h = widen8(gr[j], T());
    const Eight u = widen8(ur[j], T());
#pragma unroll
    for (int i = 0; i < 4; ++i) h.p[i] = f2_mul(silu2(h.p[i]), u.p[i]);
    float scale;
    *reinterpret_cast<uint2*>(q + 8 * v) = quantise8(h, scale, mask);
    if ((v & 15) == 0) scales[v / 16] = bf16_bits(scale);
  }
}

template <typename Kernel, typename... Args>
cudaError_t launch_dependent(Kernel kernel, dim3 blocks, dim3 threads, cudaStream_t stream,
                             const Args&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks;
  cfg.blockDim = threads;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int kVec>
cudaError_t launch_norm(const NormQuantParams& p, cudaStream_t stream) {
  const int tpr = (p.K / 8 + 32 * kVec - 1) / (32 * kVec) * 32;
  const int rows = tpr >= 128 ? 1 : 128 / tpr;
  return launch_dependent(add_rms_norm_quant_kernel<T, kVec>,
                          dim3(static_cast<unsigned>((p.M + rows - 1) / rows)), dim3(tpr, rows), stream, p);
}

template <typename T>
cudaError_t launch_norm_for(const NormQuantParams& p, cudaStream_t stream) {
  // Few rows: a row over as many threads as there are, for its latency (1 row of 4096: 2.2 us with one
  // vector a thread, 2.4 with two, 3.1 with four; 256 of 8192: 4.5, two, and 5.3, four).  Many: more work
  // a thread, but rows of 320 threads or fewer (8192 of 4096: 47.6, 40.2 and 41.2 us; of 5120: 50.9, two, and
  // 56.6, four; of 8192: 94.4, two, and 81.4, four).  512 rows is where they meet (of 4096: 4.7 us either way).
  const bool few = p.M <= 512;
  if (few && p.K <= 4096) return launch_norm<T, 1>(p, stream);
  if (p.K <= (few ? 8192 : 5120)) return launch_norm<T, 2>(p, stream);
  return launch_norm<T, 4>(p, stream);
}

}  // namespace

cudaError_t launch_add_rms_norm_quant(const NormQuantParams& p, cudaStream_t stream) {
  if (p.M == 0) return cudaSuccess;
  return p.fp16 ? launch_norm_for<__half>(p, stream) : launch_norm_for<__nv_bfloat16>(p, stream);
}

cudaError_t launch_silu_mul_quant(const SiluQuantParams& p, cudaStream_t stream) {
  if (p.M == 0) return cudaSuccess;
  const int vecs = p.I / 8;
  int tpr_log2 = 4;
  while (tpr_log2 < kSiluThreadsLog2 && kSiluVec << tpr_log2 < vecs) ++tpr_log2;
  const int64_t rows = kSiluThreads >> tpr_log2;
  const dim3 grid(static_cast<unsigned>((p.M + rows - 1) / rows),
                  (vecs + kSiluThreads * kSiluVec - 1) / (kSiluThreads * kSiluVec));
  return p.fp16 ? launch_dependent(silu_mul_quant_kernel<__half>, grid, kSiluThreads, stream, p, tpr_log2)
                : launch_dependent(silu_mul_quant_kernel<__nv_bfloat16>, grid, kSiluThreads, stream, p,
                                   tpr_log2);
}

}  // namespace fp8attn
