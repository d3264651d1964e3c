// Attention of few query rows per kv head over the paged 4-bit cache, split over the context: decode
// (one token per sequence) and short chunks of new tokens (speculative verification).
//
// The products run on the codes as they lie in the cache.  A row stands for low + step c, so
//   q . k       = step_k (q . c) + low_k sum(q)
//   sum p v     = sum (p step_v) (c - 7.5) + sum p (low_v + 7.5 step_v)
// and the steps and lowest values fold into scores and probabilities; no value is dequantised.  A 4-bit
// code in the low bits of a half is the f16 number code * 2^-24 (a subnormal, exact), four bits higher
// code * 2^-20: one mask makes a pair of operands of the tensor cores, and the powers of two are put
// into q and into the outputs.  q is exact in f16 after a power-of-two scale per row.
//
// Bound by HBM: 136 bytes of K and V for each position and kv head, read once for all of the rows of its
// query heads.  At 5.8 SM cycles per position (6.55 TB/s over 148 SMs) the math has to stay near one
// mma.sync per position, so everything stays in registers: a warp computes S^T = K q^T for 32 positions
// (A = codes, 16 positions x 16 values), turns P^T by movmatrix and adds O^T += V^T P^T (A = codes again,
// pairs of positions made by byte permutes).
//
// Work: a unit is 128 positions of one (sequence, row group, kv head), 32 for each of the CTA's four
// warps.  All units in order are cut into equal ranges, one for each resident CTA, wherever the cuts
// fall: no counters, no order that depends on timing.  A CTA's first and last piece may be parts of a
// pair; their sums go to the workspace, and a second kernel joins the parts of each cut pair in order.
// Every warp keeps a ring of its own tiles in flight (cp.async, three stages of 4.25 KB), across the ends
// of pieces.
//
// c - 7.5 is the product with c and 7.5 times the same product with ones: taken about the middle of the codes, the
// roundings of P and the cuts of the tensor cores' sums (2^-24 of each partial sum, all one way: 2e-5 of the sum
// after 512 of them) are in proportion to the values and not to their distance from the row's lowest one
// (32,768 positions: 2.1e-3 off in the 2-norm without it, 1.7e-3 with, all but the output's own rounding).
//
// Precision: scores, statistics and sums in fp32; P is rounded once, to f16 (2^-12), after its row's
// reference maximum and a power of two near the largest step of V are taken out, so it stays below 2^14.
#include <atomic>
#include <climits>

#include "common.cuh"
#include "kernels.h"

namespace fp8attn {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;               // positions per warp and unit
constexpr int kUnit = kTile * kWarps;   // positions per unit
constexpr int kStages = 3;
constexpr int kStageBytes = kTile * 136;
constexpr int kPitch = 136;             // floats between rows of the joined sums (bank spread)
constexpr float kSlack = 8.f;           // a reference maximum may lag by 2^8
constexpr float kNone = -3.402823466e38f;

template <int NT>
struct __align__(128) Smem {
  uint8_t ring[kWarps][kStages][kStageBytes];  // K rows, V rows, scales
  uint2 q[NT][8][32];                          // B operand of S^T: plane, step, lane
  float kq[8 * NT], qs[8 * NT];                // score = dot kq step + qs low
  float o[kWarps][8][kPitch];                  // a plane's sums, joined over the warps
  float m[kWarps][8], l[kWarps][8];
  int64_t scan[kWarps];
  int64_t total;
  int64_t first_unit;  // of the sequence in which the CTA's range begins
  int first_seq;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

__device__ __forceinline__ float pow2(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
__device__ __forceinline__ int exponent(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 255u) - 127; }

// A sequence's rows and visible positions; units in all.
struct Seq {
  int q_first, nq, nk, vis, tiles, groups;
  __device__ __forceinline__ int64_t units(int kvh) const {
    return static_cast<int64_t>(tiles) * groups * kvh;
  }
};

template <int NT>
__device__ __forceinline__ Seq seq_of(const Int4AttnParams& p, int s) {
  Seq q;
  if (p.cu_q != nullptr) {
    q.q_first = __ldg(p.cu_q + s);
    q.nq = __ldg(p.cu_q + s + 1) - q.q_first;
    q.nk = __ldg(p.cu_k + s + 1) - __ldg(p.cu_k + s);
    if (q.nq > p.max_q) q.nq = 0;  // the chunk kernel's
  } else {
    q.q_first = s;
    q.nq = 1;
    q.nk = __ldg(p.context_lens + s);
  }
  q.vis = max(0, min(q.nk, p.max_blocks * p.block_size));
  // a sequence without positions still has its zeros written
  q.tiles = max(1, (q.vis + kUnit - 1) / kUnit);
  q.groups = q.nq <= 0 ? 0 : (q.nq * p.group + 8 * NT - 1) / (8 * NT);
  return q;
}

// Where in the order of units a warp is.
struct Cursor {
  int seq, pair, tile;  // pair: row group * KVH + kv head
  Seq s;
};

template <int NT>
__device__ __forceinline__ void next_unit(const Int4AttnParams& p, Cursor& c) {
  if (++c.tile < c.s.tiles) return;
  c.tile = 0;
  if (++c.pair < c.s.groups * p.num_kv_heads) return;
  c.pair = 0;
  do {
    if (++c.seq >= p.num_seqs) return;
    c.s = seq_of<NT>(p, c.seq);
  } while (c.s.groups == 0);
}

// First unit of CTA i of n over u units, and the CTA that has unit x.
__device__ __forceinline__ int64_t range_begin(int64_t i, int64_t n, int64_t u) { return i * u / n; }
__device__ __forceinline__ int64_t owner(int64_t x, int64_t n, int64_t u) { return ((x + 1) * n - 1) / u; }

// The block's page of 16 positions (lane halves), -1 for none.
__device__ __forceinline__ int page_of(const Int4AttnParams& p, const Cursor& c, int warp, int lane) {
  const int pos = c.tile * kUnit + warp * kTile + (lane & 16);
  if (pos >= c.s.vis) return -1;
  const int page = ldg_keep(p.block_tables + c.seq * p.bt_stride + pos / p.block_size);
  return page >= 0 && page < p.num_blocks ? page : -1;
}

// This warp's tile of the cursor's unit into a stage; returns which halves are there (bits 0 and 1).
// Within a half (16 positions) K row i stands at row 2 (i & 3) + (i >> 2 & 1) + 8 (i >> 3), the order in which S^T's
// rows take them, and V row i at i with its 16-byte pieces changed by bit 1 of i: both are then read
// without bank conflicts.
__device__ __forceinline__ uint32_t load_tile(const Int4AttnParams& p, const Cursor& c, int page, int warp, int lane,
                                              uint32_t stage) {
  if (page >= 0) {
    const int half = lane >> 4, l = lane & 15, a = l >> 2;
    const int pos = c.tile * kUnit + warp * kTile + 16 * half;
    const int place = pos % p.block_size;
    const int kvh = c.pair % p.num_kv_heads;
    const int64_t row = (static_cast<int64_t>(page) * p.num_kv_heads + kvh) * p.block_size + place;
    const uint8_t* k = p.k_cache + row * 64 + l * 16;
    const uint8_t* v = p.v_cache + row * 64 + l * 16;
    const uint32_t kd = stage + half * 1024 + (l & 3) * 16;
    const uint32_t vd = stage + 2048 + half * 1024 + a * 64 + (((l & 3) ^ (a & 2)) * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // rows 4 i + a
      cp_async16(kd + (2 * a + (i & 1) + 8 * (i >> 1)) * 64, k + i * 256, true);
      cp_async16(vd + i * 256, v + i * 256, true);
    }
    if (l < 8) cp_async16(stage + 4096 + half * 128 + l * 16, reinterpret_cast<const uint8_t*>(p.kv_scale) + row * 8 + l * 16, true);
  }
  const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
  return (there & 1u) | (there >> 15 & 2u);
}

template <int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2) int4_decode_kernel(const Int4AttnParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(smem_raw);
  constexpr int R = 8 * NT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  // programmatic dependent of the kernel before it: nothing is read or written before that ends
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- plan: units before each sequence; thread i has sequences [i * per, (i + 1) * per)
  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += seq_of<NT>(p, s).units(p.num_kv_heads);
  int64_t before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += v;
  }
  if (lane == 31) sm.scan[warp] = before;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sm.scan[w];
    total += sm.scan[w];
  }
  before -= mine;
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);
  if (blockIdx.x == 0) {  // published for the joining kernel
    int64_t at = before;
    for (int s = s0; s < s1; ++s) {
      p.prefix[s] = at;
      at += seq_of<NT>(p, s).units(p.num_kv_heads);
    }
    if (tid == 0) p.prefix[p.num_seqs] = total;
  }
  if (blockIdx.x >= ctas) return;
  const int64_t u0 = range_begin(blockIdx.x, ctas, total), u1 = range_begin(blockIdx.x + 1, ctas, total);
  if (before <= u0 && u0 < before + mine) {
    int64_t at = before;
    int s = s0;
    for (; s < s1; ++s) {
      const int64_t n = seq_of<NT>(p, s).units(p.num_kv_heads);
      if (u0 < at + n) break;
      at += n;
    }
    sm.first_seq = s;
    sm.first_unit = at;
  }
  __syncthreads();
  Cursor now;
  now.seq = sm.first_seq;
  now.s = seq_of<NT>(p, now.seq);
  {
    const int64_t rest = u0 - sm.first_unit;
    now.pair = static_cast<int>(rest / now.s.tiles);
    now.tile = static_cast<int>(rest - static_cast<int64_t>(now.pair) * now.s.tiles);
  }

  // ---- the ring: kStages - 1 tiles in flight, and the page of the one after them
  Cursor ahead = now;
  int64_t ahead_u = u0;
  int page = page_of(p, ahead, warp, lane);
  uint32_t there = 0;  // two bits for each stage
  const uint32_t ring = smem_u32(sm.ring[warp]);
  int ahead_stage = 0;
  auto advance = [&]() {
    if (ahead_u < u1) {
      const uint32_t bits = load_tile(p, ahead, page, warp, lane, ring + ahead_stage * kStageBytes);
      there = (there & ~(3u << (2 * ahead_stage))) | bits << (2 * ahead_stage);
      ahead_stage = ahead_stage + 1 == kStages ? 0 : ahead_stage + 1;
      if (++ahead_u < u1) {
        next_unit<NT>(p, ahead);
        page = page_of(p, ahead, warp, lane);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) advance();

  int stage = 0;
  for (int64_t u = u0; u < u1;) {
    // ---- a piece: units [u, u + n) of one pair
    const int64_t n = min(u1 - u, static_cast<int64_t>(now.s.tiles - now.tile));
    const bool whole = now.tile == 0 && n == now.s.tiles;
    const int kvh = now.pair % p.num_kv_heads, rg = now.pair / p.num_kv_heads;
    const int rows = now.s.nq * p.group;  // of this kv head
    // q: the B operand of S^T, plane j by warp j.  Column (row) g, values 32 t .. 32 t + 31 in the order
    // of the codes
    if (warp < NT) {
      const int r = rg * R + 8 * warp + g;
      uint4 raw[4] = {};
      if (r < rows) {
        const int token = r / p.group;
        const uint16_t* src = p.q + (now.s.q_first + token) * p.q_row_stride +
                              (kvh * p.group + r - token * p.group) * kHeadDim + 32 * t;
#pragma unroll
        for (int w = 0; w < 4; ++w) raw[w] = ldg_keep_v4(src + 8 * w);
      }
      float amax = 0.f, sum = 0.f;
      float x[4][8];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t word[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[w][2 * i] = __uint_as_float(word[i] << 16);
          x[w][2 * i + 1] = __uint_as_float(word[i] & 0xFFFF0000u);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          amax = fmaxf(amax, fabsf(x[w][i]));
          sum += x[w][i];
        }
      }
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
      }
      // the largest value between 2^13 and 2^14; odd values, whose codes stand four bits higher, / 16
      const int e = amax > 0.f && amax < INFINITY ? max(-100, min(exponent(amax), 110)) - 13 : 0;
      const float even = pow2(-e), odd = pow2(-e - 4);
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          sm.q[warp][2 * w + b][lane] = make_uint2(pack_f16x2(x[w][2 * b] * even, x[w][2 * b + 4] * even),
                                                   pack_f16x2(x[w][2 * b + 1] * odd, x[w][2 * b + 5] * odd));
      if (t == 0) {
        sm.kq[8 * warp + g] = pow2(e) * 16777216.f * p.scale_log2;  // e + 24 <= 121
        sm.qs[8 * warp + g] = sum * p.scale_log2;
      }
    }
    __syncthreads();
    constexpr bool kHeld = NT <= 2;  // q stays in registers; else it is read from shared memory for each tile
    uint2 q[kHeld ? NT : 1][8];
    if constexpr (kHeld) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) q[j][i] = sm.q[j][i][lane];
    }
    float kq[NT][2], qs[NT][2];  // for this thread's columns 2 t and 2 t + 1
    int limit[NT][2], least = INT_MAX, most = 0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        kq[j][c] = sm.kq[8 * j + 2 * t + c];
        qs[j][c] = sm.qs[8 * j + 2 * t + c];
        const int row = rg * R + 8 * j + 2 * t + c;
        limit[j][c] = min(now.s.vis, row / p.group + now.s.nk - now.s.nq + 1);
        if (row >= rows) limit[j][c] = min(now.s.vis, rg * R / p.group + now.s.nk - now.s.nq + 1);  // no row: as the first
        least = min(least, limit[j][c]);
        most = max(most, limit[j][c]);
      }
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      least = min(least, __shfl_xor_sync(0xffffffffu, least, off));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
    }

    float o[NT][8][4], ps[NT][4], m[NT][2], l[NT][2], mid[NT][2];  // ps: sum of the rounded P step
    float v_unit = 1.f, v_limit = 0.f;  // steps of V are multiplied by v_unit (a power of two)
    int v_exp = 0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[j][c] = kNone;
        l[j][c] = mid[j][c] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) ps[j][c] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[j][i][c] = 0.f;
    }

    for (int64_t i = 0; i < n; ++i) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      const uint32_t base = ring + stage * kStageBytes;
      const uint32_t halves = there >> (2 * stage) & 3u;
      const int pos0 = (now.tile + static_cast<int>(i)) * kUnit + warp * kTile;
      advance();  // into the stage that the tile before this one has left
      if (halves != 0 && pos0 < most) {
        // ---- S^T: positions (rows g, g + 8 of each half) x query rows (columns)
        float s[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[h][j][c] = 0.f;
        uint32_t kw[2][2][4];  // half, row g or g + 8, word
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint4 k = ld_shared_v4(base + h * 1024 + (g + 8 * r) * 64 + t * 16);
            kw[h][r][0] = k.x; kw[h][r][1] = k.y; kw[h][r][2] = k.z; kw[h][r][3] = k.w;
          }
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            uint32_t a[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t y0 = kw[h][0][w] >> (8 * b), y1 = kw[h][1][w] >> (8 * b);
              a[h][0] = y0 & 0x000F000Fu;
              a[h][1] = y1 & 0x000F000Fu;
              a[h][2] = y0 & 0x00F000F0u;
              a[h][3] = y1 & 0x00F000F0u;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const uint2 qb = kHeld ? q[kHeld ? j : 0][2 * w + b] : sm.q[j][2 * w + b][lane];
              mma16816(s[0][j], a[0], qb.x, qb.y);
              mma16816(s[1][j], a[1], qb.x, qb.y);
            }
          }
        }
        // ---- scores; this thread's positions: half h, row g + 8 r stands for (g >> 1) + 4 (g & 1) + 8 r
        float sv[2][2], mv[2][2];  // step of V, and what code 7.5 stands for
        bool grow = false;
        const int mine0 = pos0 + (g >> 1) + 4 * (g & 1);
        const bool full = halves == 3u && pos0 + kTile <= least;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint2 sc = ld_shared_v2(base + 4096 + h * 128 + ((g >> 1) + 4 * (g & 1) + 8 * r) * 8);
            const float sk = __uint_as_float(sc.x << 16), lk = __uint_as_float(sc.x & 0xFFFF0000u);
            sv[h][r] = __uint_as_float(sc.y << 16);
            mv[h][r] = fmaf(7.5f, sv[h][r], __uint_as_float(sc.y & 0xFFFF0000u));
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                s[h][j][2 * r + c] = fmaf(s[h][j][2 * r + c], sk * kq[j][c], lk * qs[j][c]);
          }
        }
        if (!full) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int pos = mine0 + 16 * h + 8 * r;
              const bool held = (halves >> h & 1u) && pos < now.s.vis;
              if (!held) sv[h][r] = mv[h][r] = 0.f;
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  if (!held || pos >= limit[j][c]) s[h][j][2 * r + c] = -INFINITY;
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            grow |= sv[h][r] > v_limit;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int c = 0; c < 2; ++c) grow |= s[h][j][2 * r + c] > m[j][c] + kSlack;
          }
        if (__any_sync(0xffffffffu, grow)) {
          // ---- new references: the rows' maxima so far, and a power of two near V's largest step
          float top = fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[1][0], sv[1][1]));
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          float change = 1.f;
          if (top > v_limit && top < INFINITY) {
            const int e = max(-120, min(exponent(top), 120));
            if (v_limit > 0.f) {
              const int d = v_exp - e;
              change = d < -126 ? 0.f : pow2(d);
            }
            v_exp = e;
            v_unit = pow2(-e);
            v_limit = pow2(min(e + 6, 127));
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = fmaxf(fmaxf(s[0][j][c], s[0][j][2 + c]), fmaxf(s[1][j][c], s[1][j][2 + c]));
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              mx = fmaxf(mx, m[j][c]);
              const float f = ex2(m[j][c] - mx);
              m[j][c] = mx;
              l[j][c] *= f;
              mid[j][c] *= f;
              ps[j][c] *= f * change;
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                o[j][d][c] *= f * change;
                o[j][d][2 + c] *= f * change;
              }
            }
          }
        }
        // ---- P, its sums, and P^T step_v as the B operand of O^T
        uint32_t pb[2][NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float f = sv[h][r] * v_unit;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const float p0 = ex2(s[h][j][2 * r] - m[j][0]), p1 = ex2(s[h][j][2 * r + 1] - m[j][1]);
              l[j][0] += p0;
              l[j][1] += p1;
              mid[j][0] = fmaf(p0, mv[h][r], mid[j][0]);
              mid[j][1] = fmaf(p1, mv[h][r], mid[j][1]);
              pb[h][j][r] = transpose8x8(pack_f16x2(p0 * f, p1 * f));
            }
          }
        }
        // ---- O^T += V^T P^T: values 16 g + 2 i (rows g) and 16 g + 2 i + 1 (rows g + 8, codes four bits
        // higher) of positions t, 4 + t, 8 + t, 12 + t
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          constexpr uint32_t kOne = 0x3C003C00u;
          const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
#pragma unroll
          for (int j = 0; j < NT; ++j) mma16816(ps[j], ones, pb[h][j][0], pb[h][j][1]);
          uint2 v[4];
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4)
            v[i4] = ld_shared_v2(base + 2048 + h * 1024 + (4 * i4 + t) * 64 + (((g >> 1) ^ (t & 2)) * 16) + (g & 1) * 8);
#pragma unroll
          for (int w = 0; w < 4; ++w) {  // 4 values: half (w & 1) of word (w >> 1)
            const uint32_t sel = w & 1 ? 0x7632u : 0x5410u;
            const uint32_t x0 = __byte_perm(w < 2 ? v[0].x : v[0].y, w < 2 ? v[1].x : v[1].y, sel);
            const uint32_t x1 = __byte_perm(w < 2 ? v[2].x : v[2].y, w < 2 ? v[3].x : v[3].y, sel);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const uint32_t y0 = x0 >> (8 * b), y1 = x1 >> (8 * b);
              const uint32_t a[4] = {y0 & 0x000F000Fu, y0 & 0x00F000F0u, y1 & 0x000F000Fu, y1 & 0x00F000F0u};
#pragma unroll
              for (int j = 0; j < NT; ++j) mma16816(o[j][2 * w + b], a, pb[h][j][0], pb[h][j][1]);
            }
          }
        }
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }

    // ---- the piece's sums: the warps' parts joined through shared memory, a plane at a time
    const float unit_even = 16777216.f, unit_odd = 1048576.f, back = pow2(v_exp);
    float* part = p.partials + (2 * static_cast<int64_t>(blockIdx.x) + (u == u0 ? 0 : 1)) * (R * (kHeadDim + 2));
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], off);
          mid[j][c] += __shfl_xor_sync(0xffffffffu, mid[j][c], off);
        }
        if (g == 0) {
          sm.m[warp][2 * t + c] = m[j][c];
          sm.l[warp][2 * t + c] = l[j][c];
        }
        // value 16 g + 2 i + b at place 16 i + 2 g + b
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y0 = fmaf(fmaf(o[j][i][c], unit_even, -7.5f * ps[j][c]), back, mid[j][c]);
          const float y1 = fmaf(fmaf(o[j][i][2 + c], unit_odd, -7.5f * ps[j][c]), back, mid[j][c]);
          *reinterpret_cast<float2*>(&sm.o[warp][2 * t + c][16 * i + 2 * g]) = make_float2(y0, y1);
        }
      }
      __syncthreads();
#pragma unroll
      for (int idx = tid; idx < 8 * 64; idx += kThreads) {
        const int row = idx >> 6, place = 2 * (idx & 63);
        float mx = kNone;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm.m[w][row]);
        float y0 = 0.f, y1 = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = ex2(sm.m[w][row] - mx);
          const float2 y = *reinterpret_cast<const float2*>(&sm.o[w][row][place]);
          y0 = fmaf(y.x, f, y0);
          y1 = fmaf(y.y, f, y1);
          sum = fmaf(sm.l[w][row], f, sum);
        }
        const int in_group = 8 * j + row;
        if (whole) {
          const int r = rg * R + in_group;
          if (r < rows) {
            const int token = r / p.group;
            // 0 for a row that sees nothing
            const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
            const int value = 16 * (place >> 1 & 7) + 2 * (place >> 4);
            uint16_t* dst = p.out + (now.s.q_first + token) * p.out_row_stride +
                            (kvh * p.group + r - token * p.group) * kHeadDim + value;
            *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(y0 * inv, y1 * inv);
          }
        } else {
          *reinterpret_cast<float2*>(part + in_group * kHeadDim + place) = make_float2(y0, y1);
          if (place == 0) *reinterpret_cast<float2*>(part + R * kHeadDim + 2 * in_group) = make_float2(mx, sum);
        }
      }
      __syncthreads();
    }
    // ---- on to the next pair
    u += n;
    now.tile += static_cast<int>(n) - 1;
    if (u < u1) next_unit<NT>(p, now);
  }
  cp_async_wait<0>();
}

// Joins the parts of cut pairs: one warp for each (pair, row), parts in order.  The pairs of a sequence are
// found from the published prefix.
template <int NT>
__global__ void __launch_bounds__(128) int4_join_kernel(const Int4AttnParams p, int grid) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int R = 8 * NT;
  const int lane = threadIdx.x & 31;
  const int s = blockIdx.y;
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5);  // (row group, kv head, row)
  const Seq q = seq_of<NT>(p, s);
  const int pair = item / R, row = item - pair * R;
  if (pair >= q.groups * p.num_kv_heads) return;
  const int kvh = pair % p.num_kv_heads, rg = pair / p.num_kv_heads, r = rg * R + row;
  if (r >= q.nq * p.group) return;
  const int64_t total = p.prefix[p.num_seqs], ctas = min(static_cast<int64_t>(grid), total);
  const int64_t a = p.prefix[s] + static_cast<int64_t>(pair) * q.tiles, b = a + q.tiles;
  const int64_t c0 = owner(a, ctas, total), c1 = owner(b - 1, ctas, total);
  if (c0 == c1) return;  // one CTA had all of it
  constexpr int64_t kPart = R * (kHeadDim + 2);
  const int64_t slot0 = 2 * c0 + (a > range_begin(c0, ctas, total) ? 1 : 0);
  float mx = kNone;
  for (int64_t c = c0 + lane; c <= c1; c += 32) {
    const float* part = p.partials + (c == c0 ? slot0 : 2 * c) * kPart;
    mx = fmaxf(mx, part[R * kHeadDim + 2 * row]);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int64_t c = c0; c <= c1; ++c) {
    const float* part = p.partials + (c == c0 ? slot0 : 2 * c) * kPart;
    const float2 ml = *reinterpret_cast<const float2*>(part + R * kHeadDim + 2 * row);
    const float4 x = *reinterpret_cast<const float4*>(part + row * kHeadDim + 4 * lane);
    const float f = ex2(ml.x - mx);
    y.x = fmaf(x.x, f, y.x);
    y.y = fmaf(x.y, f, y.y);
    y.z = fmaf(x.z, f, y.z);
    y.w = fmaf(x.w, f, y.w);
    sum = fmaf(ml.y, f, sum);
  }
  const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
  const int token = r / p.group, place = 4 * lane;
  uint16_t* dst = p.out + (q.q_first + token) * p.out_row_stride +
                  (kvh * p.group + r - token * p.group) * kHeadDim + 2 * (place >> 4);
  *reinterpret_cast<__nv_bfloat162*>(dst + 16 * (place >> 1 & 7)) = __floats2bfloat162_rn(y.x * inv, y.y * inv);
  *reinterpret_cast<__nv_bfloat162*>(dst + 16 * ((place >> 1 & 7) + 1)) = __floats2bfloat162_rn(y.z * inv, y.w * inv);
}

template <int NT>
cudaError_t prepare() {
  return cudaFuncSetAttribute(int4_decode_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(sizeof(Smem<NT>)));
}

template <int NT>
int resident(int num_sms) {  // CTAs that run at once
  int per_sm = 0;
  if (prepare<NT>() != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, int4_decode_kernel<NT>, kThreads, sizeof(Smem<NT>)) !=
          cudaSuccess)
    return 0;
  return per_sm * num_sms;
}

template <int NT>
cudaError_t launch(const Int4AttnParams& p, int grid, int max_groups, cudaStream_t stream) {
  cudaError_t e = prepare<NT>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Smem<NT>);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, int4_decode_kernel<NT>, p);
  if (e != cudaSuccess) return e;
  const int64_t rows = static_cast<int64_t>(max_groups) * p.num_kv_heads * 8 * NT;
  cfg.gridDim = dim3(static_cast<unsigned>((rows + 3) / 4), static_cast<unsigned>(p.num_seqs));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, int4_join_kernel<NT>, p, grid);
}

// Planes of 8 rows in a row group: as many as the longest chunk of one kv head's rows needs, at most four.
int planes(int group, int max_q) {
  const int64_t rows = static_cast<int64_t>(group) * max_q;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : 4;
}

}  // namespace

int int4_decode_grid(int group, int max_q) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> known[kMaxDevices][4];  // by device and planes; 0: not asked yet
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  const int nt = planes(group, max_q);
  int n = known[dev][nt - 1].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    n = nt == 1 ? resident<1>(sms) : nt == 2 ? resident<2>(sms) : nt == 3 ? resident<3>(sms) : resident<4>(sms);
    known[dev][nt - 1].store(n, std::memory_order_relaxed);
  }
  return n;
}

int64_t int4_decode_workspace_bytes(int num_seqs, int group, int max_q, int grid) {
  const int64_t part = 8ll * planes(group, max_q) * (kHeadDim + 2) * 4;
  return (num_seqs + 2ll) / 2 * 16 + 2ll * grid * part;
}

cudaError_t launch_int4_decode(Int4AttnParams p, void* workspace, int grid, cudaStream_t stream) {
  const int nt = planes(p.group, p.max_q);
  p.prefix = static_cast<int64_t*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (p.num_seqs + 2ll) / 2 * 16);
  const int groups = static_cast<int>((static_cast<int64_t>(p.group) * p.max_q + 8 * nt - 1) / (8 * nt));
  switch (nt) {
    case 1: return launch<1>(p, grid, groups, stream);
    case 2: return launch<2>(p, grid, groups, stream);
    case 3: return launch<3>(p, grid, groups, stream);
    default: return launch<4>(p, grid, groups, stream);
  }
}

}  // namespace fp8attn
