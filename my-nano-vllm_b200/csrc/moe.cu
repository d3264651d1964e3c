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
//
// Bound: HBM, by the weights of the experts that are chosen (a token's 38 MB of small experts take
// 6 us, its products 0.05 us), so the weights have to stream without a pause.  Two kernels:
//
// moe_router_kernel: a cluster of 8 CTAs per few tokens; its warps share the experts' rows, the
//   logits meet in distributed shared memory, one warp per token chooses.
// moe_experts_kernel: one CTA per SM, both products.  Tokens are sorted by expert into tiles of up to
//   NT (16 or 32).  An item is 128 output columns of a tile (phase 0: 128 of gate and the same of up;
//   phase 1: 128 of the result), a unit one step of its sum, 32 KB of weights (phase 0: 128 columns of
//   K for both halves; phase 1: 256 columns of K).  A phase's units, items in order, are cut into
//   equal ranges, one per CTA, wherever the cuts fall (few tokens make few items): the parts of a cut
//   item are added, in order, by the CTA that finishes last.  CTAs take ranges by tickets, phase 0
//   first; phase 1 of a tile waits for its hidden values (a counter), which are held by ranges with
//   lower tickets, that is by CTAs that run, so the wait ends whatever else is on the GPU; meanwhile
//   the ring already holds the weights.  Sums run in an order that the choice of experts alone
//   fixes: results do not depend on timing.
//   Warps: one issues weight tiles by TMA, four gather the tokens' rows (cp.async into the same
//   swizzled layout) and scale products, two issue tcgen05 MMAs (D[128 weight rows, N tokens] per
//   128 columns of K, weights and tokens both from shared memory), eight take D from tensor memory,
//   scale and add it, and finish items.
#include <type_traits>

#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace fp8attn {
namespace {

namespace cg = cooperative_groups;

// The error word of calls that bring none.  It lives as long as the library's module, so launches in captured
// graphs may hold it, and it needs no scratch that a call would have to clear.
__device__ int g_error = 0;
__device__ __forceinline__ int* error_word(int* err) { return err != nullptr ? err : &g_error; }

// mbar_wait with its polling loop out of line: the roles' loops stay small (1 % of the layer's time).
__device__ __noinline__ bool mbar_wait_long(uint64_t* bar, uint32_t parity, int* err) {
  return mbar_wait(bar, parity, error_word(err));
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* err) {
  return mbar_try_wait(bar, parity) || mbar_wait_long(bar, parity, err);
}

// The same for a whole warp, whose lanes go on together also when a wait has given up.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, wait_for(bar, parity, err));
}

constexpr int kBlk = 128;

// A zero of either sign added to +0 is +0: sums that begin so do not depend on where a first part lay.
__device__ __forceinline__ void add4(float4& a, const float4& b) {
  a = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ __forceinline__ uint16_t f32_to_bf16(float x) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// ------------------------------------------------------------------ router
constexpr int kRouterWarps = 8;
constexpr int kRouterThreads = kRouterWarps * 32;
constexpr int kRouterCluster = 8;

// Order of the choice: larger logits first, a NaN after every number; 0 is not to be chosen.
__device__ __forceinline__ uint32_t choice_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return x == x ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 1u;  // -infinity: 0x007FFFFF
}
// The top_k largest keys by one warp, ties to the lower expert.  Lane l keeps experts l, l + 32, ..., kPer
// of them at most.  Returns the expert of place `lane`; the keys of chosen experts become 0.
template <int kPer>
__device__ __forceinline__ int choose(uint32_t (&key)[kPer], int top_k, int lane) {
  int my_id = 0;
  for (int k = 0; k < top_k; ++k) {
    uint32_t best = 0u;
#pragma unroll
    for (int j = 0; j < kPer; ++j) best = max(best, key[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    uint32_t at = 0xffffffffu;  // the lowest of the experts that have it
#pragma unroll
    for (int j = kPer - 1; j >= 0; --j)
      if (key[j] == best) at = lane + 32 * j;
    at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (static_cast<int>(at) == lane + 32 * j) key[j] = 0u;
    if (lane == k) my_id = static_cast<int>(at);
  }
  return my_id;
}

// A token's weights, and its choice with them, written by one warp: my_id is the expert of place `lane`.
__device__ __forceinline__ void write_choice(const MoeParams& p, int64_t token, const float* logits,
                                             int my_id, int lane) {
  const float chosen = logits[my_id], top = __shfl_sync(0xffffffffu, chosen, 0);
  float sum = 0.f;
  for (int e = lane; e < p.E; e += 32) sum += expf(logits[e] - top);
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

// One token's choice by one warp from logits that may be off by up to the largest of `bounds`, B; my_id: the
// expert of place `lane`.  Where no two neighbours in the order differ by 2 B or less, from the first to the
// first that is not chosen, the order is that of exact sums.  Else `open` gets the experts whose order is
// not known; returns how many.
template <int kPer>
__device__ __forceinline__ int choose_or_list(const MoeParams& p, const float* logits, const float* bounds,
                                              uint16_t* open, int& my_id, int lane) {
  uint32_t key[kPer];
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool ok = lane + 32 * j < p.E;
    key[j] = ok ? choice_key(logits[lane + 32 * j]) : 0u;
    const float b = ok ? bounds[lane + 32 * j] : 0.f;
    if (b < INFINITY) most = fmaxf(most, b);  // an infinite or NaN logit is no sum that rounding moved
  }
  const float gap = 2.f * __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
  my_id = choose<kPer>(key, p.top_k, lane);
  uint32_t rest = 0u;
#pragma unroll
  for (int j = 0; j < kPer; ++j) rest = max(rest, key[j]);
  rest = __reduce_max_sync(0xffffffffu, rest);
  const float mine = logits[my_id];
  float next = __shfl_down_sync(0xffffffffu, mine, 1);
  if (lane == p.top_k - 1)  // the best that is not chosen
    next = rest > 1u ? __uint_as_float(rest & 0x80000000u ? rest ^ 0x80000000u : ~rest) : -INFINITY;
  // places that are open against the next; a bound of 0 has no term but zeros
  const unsigned places = __ballot_sync(0xffffffffu, lane < p.top_k && gap > 0.f && mine - next <= gap);
  if (places == 0u) return 0;
  const bool listed = ((places | places << 1) >> lane & 1u) != 0u && lane < p.top_k;
  const unsigned who = __ballot_sync(0xffffffffu, listed);
  if (listed) open[__popc(who & ((1u << lane) - 1u))] = static_cast<uint16_t>(my_id);
  int count = __popc(who);
  if (places >> (p.top_k - 1) & 1u) {  // and whatever else may belong to the chosen
    const float last = __shfl_sync(0xffffffffu, mine, p.top_k - 1) - gap;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const bool more = key[j] != 0u && logits[lane + 32 * j] >= last;  // key 0: chosen, or no expert
      const unsigned them = __ballot_sync(0xffffffffu, more);
      if (more) open[count + __popc(them & ((1u << lane) - 1u))] = static_cast<uint16_t>(lane + 32 * j);
      count += __popc(them);
    }
  }
  return count;
}

// d += a . b^T: a 16 x 16, b 8 x 16 bf16.  Lane l holds a's rows l / 4 and l / 4 + 8, b's row l / 4, and
// d's rows l / 4 (d0, d1) and l / 4 + 8 (d2, d3), columns 2 (l % 4) and the next.
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 bf16 values without their signs.
__device__ __forceinline__ uint4 magnitudes(const uint4& v) {
  constexpr uint32_t kMask = 0x7FFF7FFFu;
  return make_uint4(v.x & kMask, v.y & kMask, v.z & kMask, v.w & kMask);
}

// This thread's share of x . w in fp64 (a product has 16 bits: fp32 holds it), the same columns in the same
// order whatever the row: equal rows have equal sums.
__device__ __forceinline__ double exact_part(const uint16_t* x, const uint16_t* w, int H) {
  double sum = 0.0;
  for (int v = threadIdx.x; v < H / 8; v += kRouterThreads) {
    const uint4 a = *reinterpret_cast<const uint4*>(x + 8 * v);
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(w + 8 * v));
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum += __uint_as_float(aw[i] << 16) * __uint_as_float(bw[i] << 16);
      sum += __uint_as_float(aw[i] & 0xFFFF0000u) * __uint_as_float(bw[i] & 0xFFFF0000u);
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  return sum;
}

// Cluster c: tokens 8 c .. 8 c + 7; CTA r of it: experts 16 r .. 16 r + 15, then 128 on, ...; a CTA's
// warps share the columns, 32 at a time, each lane loading 16 contiguous bytes of a row (which
// columns a product's step takes does not matter as long as both operands agree), a warp's loads
// all in flight.  Sums of 32 products in fp32, then fp64, and beside them the sums of the products'
// magnitudes, which bound what the fp32 sums may be off by.  The logits of token 8 c + r meet in CTA r, which
// chooses by them where the bound leaves no doubt, and else sums those in doubt again in fp64 (a few
// percent of the tokens of 128 experts): the experts and their order are those of exact sums.
// Bound: latency (a launch, a load from HBM, two cluster barriers, the choice): 5.6 us by itself for a token
// of 2048 columns and 128 experts, 0.8 of them for the bound, and 7.2 to 8 where some are summed again.  Two
// CTAs an SM (128 registers): the layer takes 60.1 us for 250 tokens of 60 experts, 65.3 with one.
constexpr int kRouterTokens = 8;
static_assert(kRouterTokens <= kRouterCluster, "a CTA chooses for one token at most");
// Of the magnitudes' sum, what a logit may be off by: 32 additions of at most 2^-23 each (tensor cores
// truncate) and the rounding to fp32, 2^-18 + 2^-24; the magnitudes' own sum, by 32 additions a step over up
// to 64 steps, may be 2^-12 too small.
constexpr float kLogitError = 3.9e-6f;

__global__ void __cluster_dims__(kRouterCluster, 1, 1) __launch_bounds__(kRouterThreads, 2)
    moe_router_kernel(const MoeParams p) {
  __shared__ float logits[kMoeMaxExperts], bounds[kMoeMaxExperts];
  __shared__ double part[kRouterWarps][16][kRouterTokens];
  __shared__ float part_most[kRouterWarps][16][kRouterTokens];
  __shared__ uint16_t open[kMoeMaxExperts];
  __shared__ int num_open, ids[kMoeMaxTopK];
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();  // this CTA has started: its shared memory may be written
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the counters of the next kernel
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kRouterThreads + threadIdx.x; i < p.num_counters;
       i += static_cast<int64_t>(gridDim.x) * kRouterThreads)
    p.counters[i] = 0;
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / kRouterCluster) * kRouterTokens;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int row = lane >> 2, col = 8 * (lane & 3);
  const bool real = t0 + row < p.T;
  bool started = false;
  const uint16_t* x = p.x + (t0 + row) * p.x_row_stride + col;
  for (int e0 = 16 * rank; e0 < p.E; e0 += 16 * kRouterCluster) {
    const uint16_t* w = p.router + static_cast<int64_t>(e0 + row) * p.H + col;
    const bool lo = e0 + row < p.E, hi = e0 + row + 8 < p.E;
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    float most[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int kAhead = 8;  // steps whose loads are in flight
    const int stride = 32 * kRouterWarps;
    for (int c0 = 32 * warp; c0 < p.H; c0 += kAhead * stride) {
      uint4 wl[kAhead], wh[kAhead], xv[kAhead];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        const int c = c0 + s * stride;
        wl[s] = wh[s] = xv[s] = make_uint4(0, 0, 0, 0);
        if (c < p.H) {
          if (lo) wl[s] = __ldg(reinterpret_cast<const uint4*>(w + c));
          if (hi) wh[s] = __ldg(reinterpret_cast<const uint4*>(w + 8LL * p.H + c));
          if (real) xv[s] = *reinterpret_cast<const uint4*>(x + c);
        }
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        mma_bf16(d, wl[s].x, wh[s].x, wl[s].y, wh[s].y, xv[s].x, xv[s].y);
        mma_bf16(d, wl[s].z, wh[s].z, wl[s].w, wh[s].w, xv[s].z, xv[s].w);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += d[i];
        const uint4 a = magnitudes(wl[s]), b = magnitudes(wh[s]), m = magnitudes(xv[s]);
        mma_bf16(most, a.x, b.x, a.y, b.y, m.x, m.y);
        mma_bf16(most, a.z, b.z, a.w, b.w, m.z, m.w);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      part[warp][row + 8 * (i >> 1)][2 * (lane & 3) + (i & 1)] = acc[i];
      part_most[warp][row + 8 * (i >> 1)][2 * (lane & 3) + (i & 1)] = most[i];
    }
    __syncthreads();
    if (!started) cluster.barrier_wait();
    started = true;
    const int at = threadIdx.x % (16 * kRouterTokens), e = at / kRouterTokens, t = at % kRouterTokens;
    static_assert(kRouterThreads == 2 * 16 * kRouterTokens, "half the threads for either sum");
    if (threadIdx.x < 16 * kRouterTokens) {
      double sum = 0.0;
#pragma unroll
      for (int k = 0; k < kRouterWarps; ++k) sum += part[k][e][t];
      if (e0 + e < p.E) *cluster.map_shared_rank(&logits[e0 + e], t) = static_cast<float>(sum);
    } else {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kRouterWarps; ++k) sum += part_most[k][e][t];
      if (e0 + e < p.E) *cluster.map_shared_rank(&bounds[e0 + e], t) = sum * kLogitError;
    }
    __syncthreads();
  }
  if (!started) cluster.barrier_wait();  // no experts left for this CTA
  cluster.sync();
  const int64_t token = t0 + rank;
  if (rank >= kRouterTokens || token >= p.T) return;
  int my_id = 0;
  if (warp == 0) {
    const int n = p.E <= 128  // 128 experts: 1.1 instead of 2 us
                      ? choose_or_list<4>(p, logits, bounds, open, my_id, lane)
                      : choose_or_list<kMoeMaxExperts / 32>(p, logits, bounds, open, my_id, lane);
    if (n == 0) write_choice(p, token, logits, my_id, lane);
    ids[lane] = my_id;
    if (lane == 0) num_open = n;
  }
  __syncthreads();
  const int n = num_open;
  if (n == 0) return;
  // exact sums for the open ones, a warp's share of each at a time; this CTA's `part` is free and no other
  // CTA's business
  constexpr int kSums = 64;  // experts between two barriers
  double* const exact = &part[0][0][0];  // of every expert
  double* const sums = exact + kMoeMaxExperts;
  static_assert(sizeof(part) >= (kMoeMaxExperts + kSums * kRouterWarps) * sizeof(double), "exact");
  for (int e = threadIdx.x; e < p.E; e += kRouterThreads) exact[e] = logits[e];
  for (int i0 = 0; i0 < n; i0 += kSums) {
    const int some = min(kSums, n - i0);
    for (int i = 0; i < some; ++i) {
      const double mine =
          exact_part(p.x + token * p.x_row_stride, p.router + static_cast<int64_t>(open[i0 + i]) * p.H, p.H);
      if (lane == 0) sums[i * kRouterWarps + warp] = mine;
    }
    __syncthreads();
    if (threadIdx.x < some) {
      double sum = 0.0;
#pragma unroll
      for (int k = 0; k < kRouterWarps; ++k) sum += sums[threadIdx.x * kRouterWarps + k];
      exact[open[i0 + threadIdx.x]] = sum;
      logits[open[i0 + threadIdx.x]] = static_cast<float>(sum);
    }
    __syncthreads();
  }
  // an open expert's place: how many come before it
  for (int i = warp; i < n; i += kRouterWarps) {
    const int e = open[i];
    const double mine = exact[e];
    int place = 0;
    for (int f = lane; f < p.E; f += 32) place += exact[f] > mine || (exact[f] == mine && f < e);
    place = __reduce_add_sync(0xffffffffu, place);
    if (lane == 0 && place < p.top_k) ids[place] = e;
  }
  __syncthreads();
  if (warp == 0) write_choice(p, token, logits, ids[lane], lane);
}

// ------------------------------------------------------------------ experts
constexpr int kPromoWarps = 8;  // warps 0-7
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kMmaWarps = 2;     // 9, 10: one for each of a unit's two tiles
constexpr int kLoaderWarp = 11;  // .. 14
constexpr int kLoaders = 4;
constexpr int kWarps = kLoaderWarp + kLoaders;
constexpr int kThreads = kWarps * 32;
constexpr int kDBufs = 4;
// counters: the next ticket, finished ranges of phase 1, finished items of each tile (phase 0), arrived
// parts of the item that each range leaves unfinished (by phase)
constexpr int kDoneAt = 1, kReadyAt = 2;
// Tokens per tile: 16 where an expert has 12 tokens or fewer on average, which leaves the ring more room for
// weights and the promotion threads less to do; else 32.  64 experts of 4096 x 1408, 9 tokens each: 187 us
// with 16, 195 with 32; 12 each: the same; 60 experts of 1152 x 640, 25 each: 59 us with 32.  An expert's
// tiles past the first read its weights again, and from HBM: between two readings of a weight tile the
// CTAs read more than L2 holds (8 experts of 4096 x 7168, top 2: 256 tokens read 1.75 GB for 0.70 GB of
// weights and take 311 us, 1024 tokens 5.9 GB and 1005 us).
constexpr int kFewTokens = 12;
constexpr int kMaxTiles = 896;  // at most the experts and the full tiles
static_assert(kMoeMaxExperts + kMoeMaxSlots / 32 <= kMaxTiles &&
                  kMoeMaxExperts + kFewTokens * kMoeMaxExperts / 16 <= kMaxTiles, "tiles");
int tile_tokens(int64_t T, int E, int top_k) { return T <= 16 || T * top_k <= kFewTokens * E ? 16 : 32; }

// A phase's units, items in order, are cut into equal ranges, one per CTA.  (Cutting each of few items
// into equal parts, one a range, was no faster; handing an eighth of the work out in smaller ranges,
// for SMs that get less bandwidth, was 5 to 30 % slower, since more items are cut; dealing whole
// items out in turn and cutting the rest alone was 10 % slower, since the CTAs then pause in step.)
struct Phase {
  int blocks;  // items per tile (output columns / 128)
  int steps;   // units per item
  int items;
  int units;
  int whole;   // cut between items only
  int ranges;
};
constexpr int kMaxGrid = 256;
static_assert(static_cast<uint64_t>(kMaxTiles) * 128 * 128 * (kMaxGrid + 1) < 1ull << 32, "32-bit cuts");
__device__ __forceinline__ int range_begin(const Phase& f, int r) {
  if (f.whole) return static_cast<int>(static_cast<uint32_t>(f.items) * r / f.ranges * f.steps);
  return static_cast<int>(static_cast<uint32_t>(f.units) * r / f.ranges);
}
// The range that holds unit x (not whole): the largest r with range_begin(r) <= x.
__device__ __forceinline__ int range_of(const Phase& f, int x) {
  return static_cast<int>((static_cast<uint32_t>(x + 1) * f.ranges + f.units - 1) / f.units) - 1;
}
// A range to work through: units [begin, end) of a phase, the first being step k of item (tile, blk).
struct Claim {
  int phase;  // -1: no more
  int range, begin, end;
  int tile, blk, k;
};

template <int NT>
struct __align__(1024) MoeSmem {
  static constexpr int kStages = NT == 16 ? 5 : 4;
  uint8_t w[kStages][2][kBlk * kBlk];  // weight tiles: 128 rows x 128 bytes, 128B swizzle
  uint8_t x[kStages][2][NT * kBlk];    // token tiles: NT rows x 128 bytes, 128B swizzle
  float scale[kStages][2][NT];         // activation scale * weight scale of the stage's two tiles
  float item[2][NT][kBlk];             // an item's sums (gate, up), token by token
  uint64_t w_full[kStages], x_full[kStages], empty[kStages];
  uint64_t d_full[kDBufs], d_empty[kDBufs];
  uint64_t claim_full[2], claim_empty[2];
  Claim claim[2];
  Phase phase[3];
  // promotion threads, of a cut item: the other parts have come; this CTA came last.  Two words: each is
  // written again only after a barrier that follows its last reading.
  int others_here, last;
  uint32_t tmem_base;
  int tiles;
  uint32_t tile[kMaxTiles];            // expert << 16 | index of the tile among the expert's
  uint16_t first[kMoeMaxExperts + 1];  // the expert's slots: order[first[e] .. first[e + 1])
  uint16_t order[kMoeMaxSlots];        // slots by expert
};
template <int NT>
constexpr size_t moe_smem_bytes() {
  return sizeof(MoeSmem<NT>) + 1024;
}
static_assert(moe_smem_bytes<16>() <= 227 * 1024 && moe_smem_bytes<32>() <= 227 * 1024, "smem");

__device__ __forceinline__ void promo_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// The same, and whether every thread said yes.
__device__ __forceinline__ bool promo_all(bool yes) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(yes))
      : "memory");
  return all != 0;
}

__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Adds 1 once the CTA's writes before it (its threads' by a barrier) can be seen by the GPU.
__device__ __forceinline__ void add_release(int* p) {
  asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(p) : "memory");
}
__device__ __forceinline__ int add_acq_rel(int* p) {
  int v;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// 16 bits that stay in flight until they are used (the compiler may not sink or merge the load).
__device__ __forceinline__ uint32_t load16(const uint16_t* p) {
  uint16_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t load16_fresh(const uint16_t* p) {  // written during this kernel
  uint16_t v;
  asm volatile("ld.relaxed.gpu.global.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
  return v;
}
// slot / top_k: exact for slots < 2^13 and top_k <= 32, where slot (top_k - 1) < 2^18
__device__ __forceinline__ int token_of(const MoeParams& p, int slot) {
  static_assert(kMoeMaxSlots <= 1 << 13 && kMoeMaxTopK <= 32, "token_of");
  return static_cast<int>(static_cast<uint32_t>(slot) * p.top_k_inverse >> 18);
}

// A TMA load of data that is not read again soon: first to leave L2, so that what the CTAs exchange
// stays (2-4 % faster on the batches that read 130 to 600 MB).
__device__ __forceinline__ void tma_load_once(void* dst, const CUtensorMap* map, uint64_t* bar, int x,
                                              int y) {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "l"(policy)
      : "memory");
}
// A warp's wait until *p >= want; gives up after limit_ns, recording kDevErrWaitTimeout.  Every lane has to
// have read the value: what it reads next is ordered by its own acquire (a shuffle orders no memory).
__device__ __forceinline__ bool counter_reached(const int* p, int want) {
  return __all_sync(0xffffffffu, load_acquire(p) >= want);
}
__device__ __noinline__ bool wait_counter(const int* p, int want, int* err,
                                          unsigned long long limit_ns = kWaitLimitNs) {
  unsigned long long t0 = 0;
  for (uint32_t polls = 1;; ++polls) {
    if (counter_reached(p, want)) return true;
    if ((polls & 255u) == 0) {
      const unsigned long long now = __shfl_sync(0xffffffffu, globaltimer_ns(), 0);
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > limit_ns) {
        atomicExch(error_word(err), kDevErrWaitTimeout);
        return false;
      }
    }
  }
}

// The wait by itself: lane l of one warp on counters[l].
__global__ void __launch_bounds__(32)
    counter_wait_kernel(const int* counters, int want, unsigned long long limit_ns, int* reached, int* err) {
  reached[threadIdx.x] = wait_counter(counters + threadIdx.x, want, err, limit_ns) ? 1 : 0;
}

// Slots sorted by expert (stable: results must not depend on timing), the tiles, and the two phases'
// cuts; every CTA does the same.  Scratch in the ring, which is not in use yet.
struct PlanScratch {
  uint16_t expert[kMoeMaxSlots];
  uint16_t rank[kMoeMaxSlots];             // a slot's place among its warp's slots of the expert
  uint16_t count[kWarps][kMoeMaxExperts];  // a warp's slots of an expert; zero when plan begins
  uint32_t warp_total[kMoeMaxExperts / 64];
};
template <int NT>
__device__ __forceinline__ PlanScratch& plan_scratch(MoeSmem<NT>& sm) {
  static_assert(sizeof(PlanScratch) <= 2 * sizeof(sm.w[0]), "two stages hold the scratch");
  return *reinterpret_cast<PlanScratch*>(&sm.w[0][0][0]);
}

__device__ __forceinline__ Phase make_phase(const MoeParams& p, int which, int tiles, int grid) {
  Phase f;
  if (which == 2) {  // 128 columns of a token
    f.blocks = p.H / kBlk;
    f.steps = 1;
    f.items = static_cast<int>(p.T) * f.blocks;
  } else {
    f.blocks = which == 0 ? p.I / kBlk : p.H / kBlk;
    f.steps = which == 0 ? p.H / kBlk : (p.I / kBlk + 1) / 2;
    f.items = tiles * f.blocks;
  }
  f.units = f.items * f.steps;
  // Whole items where that costs at most two units' time more than equal ranges: a cut item's parts
  // go through memory
  f.whole = (f.items + grid - 1) / grid * f.steps <= (f.units + grid - 1) / grid + 2;
  f.ranges = min(grid, f.whole ? f.items : f.units);
  return f;
}

// The range of a ticket.  Tickets: the ranges of phase 0, of phase 1, then of the weighted sums.
template <int NT>
__device__ __forceinline__ Claim make_claim(const MoeSmem<NT>& sm, int ticket) {
  Claim c = {0, ticket, 0, 0, 0, 0, 0};
  while (c.phase < 3 && c.range >= sm.phase[c.phase].ranges) c.range -= sm.phase[c.phase++].ranges;
  if (c.phase == 3) {
    c.phase = -1;
    return c;
  }
  const Phase f = sm.phase[c.phase];
  c.begin = range_begin(f, c.range);
  c.end = range_begin(f, c.range + 1);
  if (c.phase == 2) return c;
  const int item = c.begin / f.steps, some = item / f.blocks;  // some: a tile of the item's expert
  const uint32_t tile = sm.tile[some];
  const int e = static_cast<int>(tile >> 16), first = some - static_cast<int>(tile & 0xFFFFu);
  const int count = (sm.first[e + 1] - sm.first[e] + NT - 1) / NT, in = item - first * f.blocks;
  c.k = c.begin - item * f.steps;
  c.blk = in / count;
  c.tile = first + in - c.blk * count;
  return c;
}

// The lanes that have the same e as this one, among those that are ok.
__device__ __forceinline__ unsigned same_expert(int e, bool ok) {
  static_assert(kMoeMaxExperts == 512, "nine bits");
  unsigned same = __ballot_sync(0xffffffffu, ok);
#pragma unroll
  for (int b = 0; b < 9; ++b) {
    const bool one = (e >> b) & 1;
    const unsigned v = __ballot_sync(0xffffffffu, one);
    same &= one ? v : ~v;
  }
  return same;
}

template <int NT>
__device__ void plan(MoeSmem<NT>& sm, const MoeParams& p, int ticket) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int n = static_cast<int>(p.T) * p.top_k;
  PlanScratch& s = plan_scratch(sm);
  const int per = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;  // a warp's slots: [warp per, + per)
  const int lo = min(warp * per, n), hi = min(lo + per, n);
#pragma unroll 4
  for (int i = tid; i < n; i += kThreads)
    s.expert[i] = static_cast<uint16_t>(min(max(p.ids[i], 0), p.E - 1));
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    const bool ok = i < hi;
    const int e = ok ? s.expert[i] : 0;
    const unsigned same = same_expert(e, ok);
    const int base = s.count[warp][e];
    __syncwarp();
    if (ok) {
      s.rank[i] = static_cast<uint16_t>(base + __popc(same & ((1u << lane) - 1)));
      if (lane == __ffs(same) - 1) s.count[warp][e] = static_cast<uint16_t>(base + __popc(same));
    }
    __syncwarp();
  }
  __syncthreads();
  // two experts a thread, their counts side by side in 32 bits (8192 slots at most: no carry)
  const bool mine = tid < kMoeMaxExperts / 2;
  uint32_t sum = 0, before = 0;  // (slots << 16) + tiles of the experts before
  if (mine) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {  // a warp's counts -> where its slots of the expert begin
      uint32_t* c = reinterpret_cast<uint32_t*>(s.count[w]) + tid;
      const uint32_t v = *c;
      *c = sum;
      sum += v;
    }
    const uint32_t c0 = sum & 0xFFFFu, c1 = sum >> 16;
    const uint32_t own = (c0 + c1) << 16 | ((c0 + NT - 1) / NT + (c1 + NT - 1) / NT);
    uint32_t upto = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += v;
    }
    if (lane == 31) s.warp_total[warp] = upto;
    before = upto - own;
  }
  __syncthreads();
  if (mine) {
    for (int w = 0; w < warp; ++w) before += s.warp_total[w];
    const int c0 = static_cast<int>(sum & 0xFFFFu), c1 = static_cast<int>(sum >> 16);
    int slot = static_cast<int>(before >> 16), tile = static_cast<int>(before & 0xFFFFu);
    sm.first[2 * tid] = static_cast<uint16_t>(slot);
    sm.first[2 * tid + 1] = static_cast<uint16_t>(slot + c0);
    if (tid == kMoeMaxExperts / 2 - 1) sm.first[kMoeMaxExperts] = static_cast<uint16_t>(n);
    for (int j = 0; j * NT < c0; ++j) sm.tile[tile++] = static_cast<uint32_t>(2 * tid) << 16 | j;
    for (int j = 0; j * NT < c1; ++j) sm.tile[tile++] = static_cast<uint32_t>(2 * tid + 1) << 16 | j;
  } else if (warp == kWarps - 1 && lane < 3) {
    uint32_t total = 0;
    for (int w = 0; w < kMoeMaxExperts / 64; ++w) total += s.warp_total[w];
    const int tiles = static_cast<int>(total & 0xFFFFu);
    sm.phase[lane] = make_phase(p, lane, tiles, static_cast<int>(gridDim.x));
    if (lane == 0) sm.tiles = tiles;
  }
  __syncthreads();
  if (warp == kProducerWarp && lane == 0) sm.claim[0] = make_claim(sm, ticket);
  for (int i = tid; i < n; i += kThreads) {
    const int e = s.expert[i];
    sm.order[sm.first[e] + s.count[i / per][e] + s.rank[i]] = static_cast<uint16_t>(i);
  }
  // the ring's next writer is the async proxy
  fence_proxy_async_smem();
  __syncthreads();
}

// A range's place in the work; advances unit by unit.  Items run over an expert's tiles first, then over
// the column blocks, then over the experts: tiles of one expert read the same weights one after another.
template <int NT>
struct Cursor {
  int first, count;  // the expert's tiles
  int tile, blk, k;
  __device__ __forceinline__ Cursor() {}
  __device__ __forceinline__ Cursor(const MoeSmem<NT>& sm, const Claim& at)
      : tile(at.tile), blk(at.blk), k(at.k) {
    expert_of(sm, tile);
  }
  __device__ __forceinline__ void expert_of(const MoeSmem<NT>& sm, int some_tile) {
    const uint32_t t = sm.tile[some_tile];
    const int e = static_cast<int>(t >> 16);
    first = some_tile - static_cast<int>(t & 0xFFFFu);
    count = (sm.first[e + 1] - sm.first[e] + NT - 1) / NT;
  }
  __device__ __forceinline__ void next(const MoeSmem<NT>& sm, const Phase& f) {
    if (++k < f.steps) return;
    k = 0;
    if (++tile < first + count) return;
    if (++blk < f.blocks) {
      tile = first;
      return;
    }
    blk = 0;
    if (tile < sm.tiles) expert_of(sm, tile);
  }
};

template <int NT>
struct Tile {
  int expert, begin, count;  // slots order[begin .. begin + count)
  __device__ __forceinline__ Tile(const MoeSmem<NT>& sm, int tile) {
    const uint32_t t = sm.tile[tile];
    expert = static_cast<int>(t >> 16);
    begin = sm.first[expert] + static_cast<int>(t & 0xFFFFu) * NT;
    count = min(NT, sm.first[expert + 1] - begin);
  }
  __device__ __forceinline__ int columns() const { return (count + 15) & ~15; }  // the MMA's N
};

// The next range, for every warp but the producer.  False: no more.
template <int NT>
__device__ __forceinline__ bool next_claim(MoeSmem<NT>& sm, int i, int lane, int* err, Claim& claim) {
  if (!wait_warp(&sm.claim_full[i & 1], (i >> 1) & 1, err)) return false;
  claim = sm.claim[i & 1];
  __syncwarp();
  if (lane == 0) mbar_arrive(&sm.claim_empty[i & 1]);
  return claim.phase >= 0;
}

template <int NT>
__device__ void produce(MoeSmem<NT>& sm, const MoeParams& p, const CUtensorMap* tm13,
                        const CUtensorMap* tm2) {
  constexpr int kStages = MoeSmem<NT>::kStages;
  uint32_t r = 0;
  bool ok = true;
  int ticket = 0;
  for (int i = 0;; ++i) {
    Claim claim = sm.claim[0];  // the first one was made with the plan
    if (i > 0) {
      claim = make_claim(sm, ticket);
      ok = ok && wait_for(&sm.claim_empty[i & 1], ((i >> 1) & 1) ^ 1, p.err);
      if (!ok) claim.phase = -1;
      sm.claim[i & 1] = claim;
    }
    mbar_arrive(&sm.claim_full[i & 1]);
    const int ph = claim.phase;
    if (ph < 0) break;
    if (ph == 2) {  // nothing to load
      ticket = atomicAdd(p.counters, 1);
      continue;
    }
    const Phase f = sm.phase[ph];
    Cursor<NT> c(sm, claim);
    for (int u = claim.begin; u < claim.end && ok; ++u, ++r, c.next(sm, f)) {
      // the next ticket: its latency hides behind this range, whose first half lets a CTA that starts
      // late have its turn (one that held two ranges of a phase would take twice as long)
      if (u == claim.begin + (claim.end - claim.begin) / 2) ticket = atomicAdd(p.counters, 1);
      const int stage = r % kStages;
      const int expert = static_cast<int>(sm.tile[c.tile] >> 16);
      if (!wait_for(&sm.empty[stage], ((r / kStages) & 1) ^ 1, p.err)) {
        ok = false;
        break;
      }
      if (ph == 0) {
        mbar_arrive_expect_tx(&sm.w_full[stage], 2 * kBlk * kBlk);
        const int row = expert * 2 * p.I + c.blk * kBlk;
        tma_load_once(sm.w[stage][0], tm13, &sm.w_full[stage], c.k * kBlk, row);
        tma_load_once(sm.w[stage][1], tm13, &sm.w_full[stage], c.k * kBlk, row + p.I);
      } else {
        const bool two = (2 * c.k + 1) * kBlk < p.I;
        mbar_arrive_expect_tx(&sm.w_full[stage], (two ? 2 : 1) * kBlk * kBlk);
        const int row = expert * p.H + c.blk * kBlk;
        tma_load_once(sm.w[stage][0], tm2, &sm.w_full[stage], 2 * c.k * kBlk, row);
        if (two) tma_load_once(sm.w[stage][1], tm2, &sm.w_full[stage], (2 * c.k + 1) * kBlk, row);
      }
    }
  }
  // After a wait that gave up: the copies still in flight land before the CTA ends.
  for (uint32_t u = r < kStages ? 0 : r - kStages; !ok && u < r; ++u)
    wait_for(&sm.w_full[u % kStages], (u / kStages) & 1, p.err);
}

// One of the gather warps: its share of the units, round robin.  A unit's copies and scales are in
// flight while the next one's are issued; the two sets of scale registers alternate, since a copy of a
// register waits for its load (measured: 470 instead of 190 us for 64 tokens).
template <int NT>
struct Gather {
  static constexpr int kStages = MoeSmem<NT>::kStages;
  static constexpr int kPer = (NT + 31) / 32;  // tokens a lane scales

  struct Unit {
    int stage = -1;  // -1: none in flight
    uint32_t act[2][kPer], weight[2];  // bf16 bits: lane's activation scales and the weight's, by tile
  };

  MoeSmem<NT>& sm;
  const MoeParams& p;
  const int which, lane, kc1, kc2;
  Phase f;
  Cursor<NT> c;
  int u = 0, end = 0, ph = 0, claims = 0, ready = -1;
  uint32_t r = 0;
  bool ok = true;

  __device__ Gather(MoeSmem<NT>& s, const MoeParams& q, int w, int l)
      : sm(s), p(q), which(w), lane(l), kc1(q.H / kBlk), kc2(q.I / kBlk) {}

  // The unit's tiles are complete: newer: another unit's copies were issued after its own.
  __device__ __forceinline__ void finish(Unit& unit, bool newer) {
    if (unit.stage < 0) return;
#pragma unroll
    for (int h = 0; h < kPer; ++h)
      if (lane + 32 * h < NT) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
          sm.scale[unit.stage][s][lane + 32 * h] =
              __uint_as_float(unit.act[s][h] << 16) * __uint_as_float(unit.weight[s] << 16);
      }
    if (newer) {
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    fence_proxy_async_smem();  // the tensor cores read the rows through the async proxy
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.x_full[unit.stage]);
    unit.stage = -1;
  }

  // To this warp's next unit; false: no more.  Whatever may have to wait lets the unit in flight go
  // first: the wait may depend on it.
  __device__ __forceinline__ bool advance(Unit& flying) {
    for (;;) {
      while (u == end) {
        Claim claim;
        finish(flying, false);
        if (!next_claim(sm, claims++, lane, p.err, claim)) return false;
        ph = claim.phase;
        if (ph == 2) continue;
        f = sm.phase[ph];
        u = claim.begin;
        end = claim.end;
        c = Cursor<NT>(sm, claim);
        ready = -1;
      }
      if (static_cast<int>(r % kLoaders) == which) return true;
      step();
    }
  }
  __device__ __forceinline__ void step() {
    ++u;
    ++r;
    c.next(sm, f);
  }

  // Issues the next unit into `mine`, then completes `other`.
  __device__ __forceinline__ bool run(Unit& mine, Unit& other) {
    if (!advance(other)) return false;
    const int stage = r % kStages;
    if (ok && ph == 1 && c.tile != ready) {  // the tile's hidden values: written by other CTAs
      const int* counter = p.counters + kReadyAt + c.tile;
      if (!counter_reached(counter, kc2)) {
        finish(other, false);
        ok = wait_counter(counter, kc2, p.err);
      }
      ready = c.tile;
    }
    if (ok && !__all_sync(0xffffffffu, mbar_test(&sm.empty[stage], ((r / kStages) & 1) ^ 1))) {
      finish(other, false);
      ok = wait_warp(&sm.empty[stage], ((r / kStages) & 1) ^ 1, p.err);
    }
    if (ok) {  // else: the others stop by themselves, their waits on this stage are bounded
      issue(mine, stage);
      finish(other, true);
    }
    step();
    return true;
  }

  __device__ __forceinline__ void issue(Unit& unit, int stage) {
    unit.stage = stage;
    const Tile<NT> t(sm, c.tile);
    const int subs = ph == 0 ? 1 : (2 * c.k + 1 < kc2 ? 2 : 1);
    if (ph == 0) {
      const uint16_t* ws = p.w13_scale + (static_cast<int64_t>(t.expert) * 2 * kc2 + c.blk) * kc1 + c.k;
      unit.weight[0] = load16(ws);
      unit.weight[1] = load16(ws + static_cast<int64_t>(kc2) * kc1);
    } else {
      const uint16_t* ws = p.w2_scale + (static_cast<int64_t>(t.expert) * kc1 + c.blk) * kc2 + 2 * c.k;
      unit.weight[0] = load16(ws);
      unit.weight[1] = subs == 2 ? load16(ws + 1) : 0u;
    }
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      const int m = lane + 32 * h;
      unit.act[0][h] = unit.act[1][h] = 0u;
      if (m < t.count) {
        const int slot = sm.order[t.begin + m];
        if (ph == 0) {
          unit.act[0][h] = load16(p.x_scale + static_cast<int64_t>(token_of(p, slot)) * kc1 + c.k);
          unit.act[1][h] = unit.act[0][h];
        } else {
          const uint16_t* hs = p.h_scale + static_cast<int64_t>(slot) * kc2 + 2 * c.k;
          unit.act[0][h] = load16_fresh(hs);
          if (subs == 2) unit.act[1][h] = load16_fresh(hs + 1);
        }
      }
    }
    // rows: 8 lanes copy a row's 128 bytes; rows past the tile's tokens are zeros
    const int rows = t.columns(), chunk = lane & 7;
    for (int m = lane >> 3; m < rows; m += 4) {
      const bool real = m < t.count;
      const int slot = real ? sm.order[t.begin + m] : 0;
      const uint8_t* src =
          ph == 0 ? p.xq + static_cast<int64_t>(token_of(p, slot)) * p.xq_row_stride + c.k * kBlk
                  : p.hq + static_cast<int64_t>(slot) * p.I + 2 * c.k * kBlk;
      const uint32_t at = m * kBlk + ((chunk ^ (m & 7)) << 4);
      cp_async16(smem_u32(sm.x[stage][0]) + at, src + chunk * 16, real);
      if (subs == 2) cp_async16(smem_u32(sm.x[stage][1]) + at, src + kBlk + chunk * 16, real);
    }
    cp_async_commit();
  }

  __device__ void run_all() {
    Unit a, b;
    while (run(a, b) && run(b, a)) {
    }
    finish(a, false);
    finish(b, false);
  }
};

// MMA issuer `which`: that one of each unit's two tiles.  An MMA holds its issuing thread for about 100
// cycles: one thread for both tiles took 0.83 us a unit, 39 GB/s an SM, and paced the whole kernel.
template <int NT>
__device__ void multiply(MoeSmem<NT>& sm, const MoeParams& p, int which, int lane) {
  constexpr int kStages = MoeSmem<NT>::kStages;
  const uint32_t tmem = sm.tmem_base + which * NT;
  // descriptors of stage 0; a stage and 32 bytes of K add to the start address / 16
  const uint64_t w0 = tc::smem_desc(smem_u32(sm.w[0][which]), 16, 1024, tc::kSw128);
  const uint64_t x0 = tc::smem_desc(smem_u32(sm.x[0][0]), 16, 1024, tc::kSw128);
  uint32_t r = 0;
  bool ok = true;
  Claim claim;
  for (int i = 0; next_claim(sm, i, lane, p.err, claim); ++i) {
    const int ph = claim.phase;
    if (lane == 0 && ph < 2) {
      const Phase f = sm.phase[ph];
      Cursor<NT> c(sm, claim);
      const uint64_t xs = x0 + (ph == 1 ? which * (sizeof(sm.x[0][0]) >> 4) : 0);
      int tile = -1;
      uint32_t idesc = 0;
      for (int u = claim.begin; u < claim.end && ok; ++u, ++r, c.next(sm, f)) {
        const int stage = r % kStages, buf = r % kDBufs;
        if (c.tile != tile) {
          tile = c.tile;
          idesc = tc::idesc_e4m3(kBlk, Tile<NT>(sm, tile).columns(), false, false);
        }
        ok = wait_for(&sm.w_full[stage], (r / kStages) & 1, p.err) &&
             wait_for(&sm.x_full[stage], (r / kStages) & 1, p.err) &&
             wait_for(&sm.d_empty[buf], ((r / kDBufs) & 1) ^ 1, p.err);
        if (!ok) break;
        tc::fence_after_sync();
        if (which == 0 || ph == 0 || (2 * c.k + 1) * kBlk < p.I) {
          const uint64_t wd = w0 + stage * (sizeof(sm.w[0]) >> 4), xd = xs + stage * (sizeof(sm.x[0]) >> 4);
#pragma unroll
          for (int ks = 0; ks < kBlk / 32; ++ks)
            tc::mma_f8_plain(tmem + buf * 2 * NT, wd + static_cast<uint64_t>(2 * ks),
                             xd + static_cast<uint64_t>(2 * ks), idesc, ks > 0 ? 1u : 0u);
        }
        tc::commit(&sm.d_full[buf]);
        tc::commit(&sm.empty[stage]);
      }
    }
    __syncwarp();
  }
}

// acc[j] += d[j] * s[j] over one of the unit's two tiles: this thread's weight row, `groups` groups of 8
// tokens from column `col`.
template <int NT>
__device__ __forceinline__ void scale_add(float (&acc)[NT / 2], uint32_t taddr, const float* s,
                                          int groups) {
  constexpr int kBatch = NT / 16 < 2 ? 1 : 2;  // loads in flight together; more of them spill
#pragma unroll
  for (int q0 = 0; q0 < NT / 16; q0 += kBatch) {
    if (q0 >= groups) break;
    float d[kBatch][8];
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
      if (q0 + q < groups) tc::ld8(taddr + 8 * (q0 + q), d[q]);
    tc::wait_ld();
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
      if (q0 + q < groups) {
        const float4 a = *reinterpret_cast<const float4*>(s + 8 * (q0 + q));
        const float4 b = *reinterpret_cast<const float4*>(s + 8 * (q0 + q) + 4);
        const float sc[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc[8 * (q0 + q) + j] = fmaf(d[q][j], sc[j], acc[8 * (q0 + q) + j]);
      }
  }
}

// The promotion warps: warp w has tensor-memory lanes 32 (w % 4) .. + 31 (an item's output columns)
// and half w / 4 of the tile's tokens.
template <int NT>
__device__ void promote(MoeSmem<NT>& sm, const MoeParams& p, int warp, int lane) {
  constexpr int kStages = MoeSmem<NT>::kStages;
  constexpr int kHalf = NT / 2;
  const int quad = warp & 3, half = warp >> 2, tid = warp * 32 + lane;
  const int col = 32 * quad + lane;  // output column of the item
  const uint32_t tmem = sm.tmem_base + (static_cast<uint32_t>(32 * quad) << 16);
  const int kc2 = p.I / kBlk;
  int* const ready = p.counters + kReadyAt;
  int* const part_count = ready + kMaxTiles;  // [2][grid]
  uint32_t r = 0;
  bool ok = true;
  Claim claim;
  for (int i = 0; promo_all(next_claim(sm, i, lane, p.err, claim)); ++i) {
    const int ph = claim.phase, range = claim.range, begin = claim.begin, end = claim.end;
    const Phase f = sm.phase[ph];
    if (ph == 2) {
      // ---- weighted sums, once phase 1 has ended: its ranges are held by CTAs that run
      ok = ok && wait_counter(p.counters + kDoneAt, sm.phase[1].ranges, p.err);
      for (int item = begin + warp; item < end && ok; item += kPromoWarps) {
        const int64_t token = item / f.blocks;
        const int at = (item - static_cast<int>(token) * f.blocks) * kBlk + lane * 4;
        const float* y = p.y + token * p.top_k * p.H + at;
        const float* w = p.weights + token * p.top_k;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < p.top_k; k0 += 8) {  // eight slots' loads in flight
          float4 v[8];
          float c[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const bool have = k0 + k < p.top_k;
            v[k] = have ? __ldcg(reinterpret_cast<const float4*>(y + static_cast<int64_t>(k0 + k) * p.H))
                        : make_float4(0.f, 0.f, 0.f, 0.f);
            c[k] = have ? __ldg(w + k0 + k) : 0.f;
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            acc.x = fmaf(c[k], v[k].x, acc.x);
            acc.y = fmaf(c[k], v[k].y, acc.y);
            acc.z = fmaf(c[k], v[k].z, acc.z);
            acc.w = fmaf(c[k], v[k].w, acc.w);
          }
        }
        const uint32_t lo = f32_to_bf16(acc.x) | static_cast<uint32_t>(f32_to_bf16(acc.y)) << 16;
        const uint32_t hi = f32_to_bf16(acc.z) | static_cast<uint32_t>(f32_to_bf16(acc.w)) << 16;
        *reinterpret_cast<uint2*>(p.out + token * p.out_row_stride + at) = make_uint2(lo, hi);
      }
      continue;
    }
    Cursor<NT> c(sm, claim);
    int u = begin;
    while (u < end) {
      // ---- one item, or the part of it that this range holds
      const Tile<NT> t(sm, c.tile);
      const int groups = t.columns() / 16, m0 = half * 8 * groups;  // tokens m0 .. m0 + 8 groups - 1
      const int item_begin = u - c.k;
      const int stop = min(end, item_begin + f.steps);
      const bool cut = u != item_begin || stop != item_begin + f.steps;
      const int tile = c.tile, blk = c.blk;
      float g[kHalf], v[kHalf];
#pragma unroll
      for (int j = 0; j < kHalf; ++j) g[j] = v[j] = 0.f;
      const bool at_head = u != item_begin;
      // a cut item's parts: those of ranges r0 .. r1
      const int r0 = cut ? range_of(f, item_begin) : 0;
      const int r1 = cut ? range_of(f, item_begin + f.steps - 1) : 0;
      int* const arrived = part_count + ph * gridDim.x + r0;
      int others = 0;
      for (; u < stop; ++u, ++r, c.next(sm, f)) {
        const int stage = r % kStages, buf = r % kDBufs;
        // whoever begins an item usually comes last to it: are the other parts there already?
        if (u == stop - 1 && cut && !at_head && tid == 0) others = load_acquire(arrived);
        ok = ok && wait_warp(&sm.x_full[stage], (r / kStages) & 1, p.err) &&
             wait_warp(&sm.d_full[buf], (r / kDBufs) & 1, p.err);
        if (!ok) continue;  // and on through the barriers, which need every warp
        tc::fence_after_sync();
        const uint32_t d = tmem + buf * 2 * NT + m0;
        scale_add<NT>(g, d, &sm.scale[stage][0][m0], groups);
        if (ph == 0) {
          scale_add<NT>(v, d + NT, &sm.scale[stage][1][m0], groups);
        } else if (2 * c.k + 1 < kc2) {
          scale_add<NT>(g, d + NT, &sm.scale[stage][1][m0], groups);
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm.d_empty[buf]);
          mbar_arrive(&sm.empty[stage]);
        }
      }
      // ---- the item's sums, token by token: through shared memory, and, of a cut item, through global
      // memory, where the CTA that comes last adds the parts, in order
      constexpr int kPart = NT * kBlk;  // floats; phase 0 has two of them (gate, up)
      float* const parts = p.parts[ph];
      const int size = ph == 0 ? 2 * kPart : kPart;
      float* const mine = parts + (2 * static_cast<int64_t>(range) + (at_head ? 0 : 1)) * size;
      float* to = at_head ? mine : &sm.item[0][0][0];
      if (tid == 0) sm.others_here = others == r1 - r0;
      bool here;  // part 0 in shared memory, the others complete
#pragma unroll 1
      for (;;) {  // once, or, for the beginner of an item whose other parts are not there, twice
#pragma unroll
        for (int j = 0; j < kHalf; ++j)
          if (j < 8 * groups) {
            to[(m0 + j) * kBlk + col] = g[j];
            if (ph == 0) to[kPart + (m0 + j) * kBlk + col] = v[j];
          }
        promo_sync();
        here = to != mine && (!cut || sm.others_here);
        if (here || to == mine) break;
        to = mine;
      }
      if (!here) {
        if (tid == 0) sm.last = add_acq_rel(arrived) == r1 - r0;
        promo_sync();
        if (!sm.last) continue;
      }
      // kLanes lanes take a token: lane l columns 4 (l + kLanes i) .. + 3. With up to 32 tokens an item, two
      // tokens a warp halve the turns (250 tokens, 60 experts, top 6: 63.1 to 60.1 us); with few, a warp a
      // token has the shorter chain (1 token: 26.8 us against 27.2; 16 tokens: 78.1 against 78.9).
      constexpr int kLanes = NT == 16 ? 32 : 16, kQuads = 32 / kLanes, kTokens = kPromoWarps * 32 / kLanes;
      constexpr int kTogether = NT == 16 ? 4 : 2;  // parts whose loads are in flight together
      const int at = 4 * (lane % kLanes);
#pragma unroll 1  // one turn at a time: unrolled by two, the larger code cost 2 to 7 %
      for (int first = warp * (32 / kLanes); first < t.count; first += kTokens) {
        const int m = min(first + lane / kLanes, t.count - 1);  // an odd last token twice, with equal results
        float4 a[kQuads], b[kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          a[i] = b[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (here) {
            add4(a[i], *reinterpret_cast<const float4*>(&sm.item[0][m][at + 4 * kLanes * i]));
            if (ph == 0) add4(b[i], *reinterpret_cast<const float4*>(&sm.item[1][m][at + 4 * kLanes * i]));
          }
        }
#pragma unroll 1
        for (int q0 = here ? r0 + 1 : r0; cut && q0 <= r1; q0 += kTogether) {
          float4 pa[kTogether][kQuads], pb[kTogether][kQuads];
#pragma unroll
          for (int d = 0; d < kTogether; ++d) {
            const float* part = parts + (2 * static_cast<int64_t>(q0 + d) + (q0 + d == r0 ? 1 : 0)) * size +
                                m * kBlk + at;
#pragma unroll
            for (int i = 0; i < kQuads; ++i) {
              pa[d][i] = pb[d][i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (q0 + d <= r1) {
                pa[d][i] = __ldcg(reinterpret_cast<const float4*>(part + 4 * kLanes * i));
                if (ph == 0) pb[d][i] = __ldcg(reinterpret_cast<const float4*>(part + kPart + 4 * kLanes * i));
              }
            }
          }
#pragma unroll
          for (int d = 0; d < kTogether; ++d)
#pragma unroll
            for (int i = 0; i < kQuads; ++i) {
              add4(a[i], pa[d][i]);
              add4(b[i], pb[d][i]);
            }
        }
        const int64_t slot = sm.order[t.begin + m];
        if (ph == 1) {
          float* const y = p.y + slot * p.H + blk * kBlk + at;
#pragma unroll
          for (int i = 0; i < kQuads; ++i) __stcg(reinterpret_cast<float4*>(y + 4 * kLanes * i), a[i]);
        } else {
          // h = silu(gate) up, quantised over the item's 128 columns
          float h[4 * kQuads], most = 0.f;
#pragma unroll
          for (int i = 0; i < kQuads; ++i) {
            f2_unpack(f2_mul(silu2(f2_pack(a[i].x, a[i].y)), f2_pack(b[i].x, b[i].y)), h[4 * i], h[4 * i + 1]);
            f2_unpack(f2_mul(silu2(f2_pack(a[i].z, a[i].w)), f2_pack(b[i].z, b[i].w)), h[4 * i + 2],
                      h[4 * i + 3]);
          }
#pragma unroll
          for (int i = 0; i < 4 * kQuads; ++i) most = fmaxf(most, fabsf(h[i]));  // NaN left out
#pragma unroll
          for (int off = kLanes < 32 ? kLanes / 2 : 0; off > 0; off >>= 1)
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
          if (kLanes == 32) most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
          const float scale = divide_by_scale(h, most);
          uint8_t* const q = p.hq + slot * p.I + blk * kBlk + at;
#pragma unroll
          for (int i = 0; i < kQuads; ++i)
            *reinterpret_cast<uint32_t*>(q + 4 * kLanes * i) =
                f32x2_to_e4m3x2(h[4 * i], h[4 * i + 1]) | (f32x2_to_e4m3x2(h[4 * i + 2], h[4 * i + 3]) << 16);
          if (at == 0) p.h_scale[slot * kc2 + blk] = f32_to_bf16(scale);
        }
      }
      promo_sync();  // what was written is complete; the shared item is free again
      if (ph == 0 && tid == 0) add_release(ready + tile);
    }
    if (ph == 1) {
      promo_sync();
      if (tid == 0) add_release(p.counters + kDoneAt);
    }
  }
}

template <int NT>
__global__ void __launch_bounds__(kThreads, 1)
    moe_experts_kernel(const __grid_constant__ CUtensorMap tm13, const __grid_constant__ CUtensorMap tm2,
                       const MoeParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  MoeSmem<NT>& sm = *reinterpret_cast<MoeSmem<NT>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr uint32_t kColumns = kDBufs * 2 * NT;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < MoeSmem<NT>::kStages; ++i) {
      mbar_init(&sm.w_full[i], 1);
      mbar_init(&sm.x_full[i], 1);
      mbar_init(&sm.empty[i], kMmaWarps + kPromoWarps);
    }
    for (int i = 0; i < kDBufs; ++i) {
      mbar_init(&sm.d_full[i], kMmaWarps);
      mbar_init(&sm.d_empty[i], kPromoWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.claim_full[i], 1);
      mbar_init(&sm.claim_empty[i], kPromoWarps + kMmaWarps + kLoaders);
    }
    fence_mbar_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tensormap(&tm13);
    prefetch_tensormap(&tm2);
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(&sm.tmem_base, kColumns);
    tc::tmem_relinquish();
  }
  for (int i = threadIdx.x; i < kWarps * kMoeMaxExperts / 2; i += kThreads)
    reinterpret_cast<uint32_t*>(plan_scratch(sm).count)[i] = 0;
  // launched as a programmatic dependent of the router: its choice is read only when it has ended
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int ticket = 0;
  if (warp == kProducerWarp && lane == 0) ticket = atomicAdd(p.counters, 1);
  tc::fence_before_sync();
  plan<NT>(sm, p, ticket);  // barriers of the whole CTA
  tc::fence_after_sync();
  if (warp == kProducerWarp) {
    if (lane == 0) produce<NT>(sm, p, &tm13, &tm2);
    __syncwarp();
  } else if (warp >= kMmaWarp && warp < kLoaderWarp) {
    multiply<NT>(sm, p, warp - kMmaWarp, lane);
  } else if (warp >= kLoaderWarp) {
    Gather<NT>(sm, p, warp - kLoaderWarp, lane).run_all();
  } else {
    promote<NT>(sm, p, warp, lane);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == kMmaWarp) tc::tmem_dealloc(sm.tmem_base, kColumns);
}

int moe_grid(int num_sms) { return num_sms < kMaxGrid ? num_sms : kMaxGrid; }

template <int NT>
cudaError_t launch_experts(const MoeParams& p, int num_sms, cudaStream_t stream) {
  CUtensorMap tm13, tm2;
  if (!make_rows_map(&tm13, p.w13, static_cast<int64_t>(p.E) * 2 * p.I, p.H, p.H, kBlk) ||
      !make_rows_map(&tm2, p.w2, static_cast<int64_t>(p.E) * p.H, p.I, p.I, kBlk))
    return cudaErrorInvalidValue;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  constexpr int smem = static_cast<int>(moe_smem_bytes<NT>());
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(moe_experts_kernel<NT>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(moe_grid(num_sms));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, moe_experts_kernel<NT>, tm13, tm2, p);
}

cudaError_t launch_router(const MoeParams& p, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.T + kRouterTokens - 1) / kRouterTokens) * kRouterCluster);
  cfg.blockDim = dim3(kRouterThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, moe_router_kernel, p);
}

}  // namespace

cudaError_t launch_counter_wait(const int* counters, int want, unsigned long long limit_ns, int* reached, int* err,
                                cudaStream_t stream) {
  counter_wait_kernel<<<1, 32, 0, stream>>>(counters, want, limit_ns, reached, err);
  return cudaGetLastError();
}

cudaError_t moe_error_word(void** word) { return cudaGetSymbolAddress(word, g_error); }

int64_t moe_layout(MoeParams& p, void* workspace, int num_sms) {
  uint8_t* const base = static_cast<uint8_t*>(workspace);
  int64_t off = 0;
  auto take = [&](auto*& ptr, int64_t bytes) {
    if (base != nullptr && ptr == nullptr)
      ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(base + off);
    off += (bytes + 255) / 256 * 256;
  };
  const int64_t n = p.T * p.top_k, part = static_cast<int64_t>(tile_tokens(p.T, p.E, p.top_k)) * kBlk * 4;
  const int64_t ranges = moe_grid(num_sms);
  p.num_counters = kReadyAt + kMaxTiles + 2 * ranges;
  p.top_k_inverse = ((1u << 18) + p.top_k - 1) / p.top_k;
  take(p.counters, p.num_counters * 4);
  take(p.ids, n * 4);  // where the caller gives none
  take(p.weights, n * 4);
  take(p.hq, n * p.I);
  take(p.h_scale, n * (p.I / kBlk) * 2);
  take(p.y, n * p.H * 4);
  take(p.parts[0], 2 * ranges * 2 * part);
  take(p.parts[1], 2 * ranges * part);
  return off;
}

cudaError_t launch_moe(const MoeParams& p, int num_sms, cudaStream_t stream) {
  if (p.T == 0) return cudaSuccess;
  const cudaError_t e = launch_router(p, stream);
  if (e != cudaSuccess) return e;
  return tile_tokens(p.T, p.E, p.top_k) == 16 ? launch_experts<16>(p, num_sms, stream)
                                : launch_experts<32>(p, num_sms, stream);
}

}  // namespace fp8attn
