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
// Every warp keeps two of its own tiles of 4.25 KB in flight (TMA, 64B swizzle, one lane issues), across the ends
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

#include "int4_attention.cuh"

namespace fp8attn {
namespace {

// The error word of these kernels' launches: it lives as long as the library's module, so that captured graphs may
// hold its address.
__device__ int g_error = 0;

#ifndef INT4_W
#define INT4_W 4
#define INT4_S 3
#define INT4_C 3
#endif
constexpr int kWarps = INT4_W;          // that compute; one more loads
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kTile = 32;               // positions per warp and unit
constexpr int kUnit = kTile * kWarps;   // positions per unit
constexpr int kParts = kUnit / 16;      // parts of a unit that lie in one page each
constexpr int kStages = INT4_S;
constexpr int kPitch = 136;             // floats between rows of the joined sums (bank spread)
constexpr float kSlack = 8.f;           // a reference maximum may lag by 2^8

template <int NT>
struct __align__(1024) Smem {
  uint8_t k[kStages][kUnit * 64];  // TMA tiles of 64-byte rows, 64B swizzle: bits 1 and 2 of a row's number
  uint8_t v[kStages][kUnit * 64];  // change the place of its 16-byte pieces
  uint2 scale[kStages][kUnit];
  uint2 q[NT][8][32];              // B operand of S^T: plane, step, lane
  float kq[8 * NT], qs[8 * NT];    // score = dot kq step + qs low
  float o[kWarps][8][kPitch];      // a plane's sums, joined over the warps
  float m[kWarps][8], l[kWarps][8];
  uint64_t full[kStages], empty[kStages];
  uint32_t there[kStages];         // which parts of the stage's unit are in pages of the cache
  int64_t scan[kWarps + 1];
  int64_t first_unit;              // of the sequence in which the CTA's range begins
  int first_seq;
};

// The computing warps alone.
__device__ __forceinline__ void sync_compute() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b: no registers to be cleared first.
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// w >> 8 on the multiply pipe (by = 2^24, in a register so that it stays a product): the unpacking's masks keep
// the integer pipe busier than anything else.
__device__ __forceinline__ uint32_t shift8(uint32_t w, uint32_t by) {
  uint32_t d;
  d = w >> 8; (void)by;
  return d;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// Four 8 x 8 matrices of 16-bit elements, transposed: lanes 8 i .. 8 i + 7 give the rows of matrix i.
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// A sequence's rows and visible positions; units in all.
struct Seq {
  int q_first, nq, nk, vis, tiles, groups;
  __device__ __forceinline__ int64_t units(int kvh) const {
    return static_cast<int64_t>(tiles) * groups * kvh;
  }
};

template <int R>
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
  q.groups = q.nq <= 0 ? 0 : (q.nq * p.group + R - 1) / R;
  return q;
}

// Where in the order of units a warp is.
struct Cursor {
  int seq, pair, tile;  // pair: row group * KVH + kv head
  Seq s;
};

template <int R>
__device__ __forceinline__ void next_pair(const Int4AttnParams& p, Cursor& c) {
  c.tile = 0;
  if (++c.pair < c.s.groups * p.num_kv_heads) return;
  c.pair = 0;
  do {
    if (++c.seq >= p.num_seqs) return;
    c.s = seq_of<R>(p, c.seq);
  } while (c.s.groups == 0);
}

// The loading warp: lane i looks up the page of part i of each unit, and the lanes at which a TMA box begins load it
// (box_rows positions: K, V and scales).  The pages of the next unit are looked up before this one's stage is waited
// for.
template <int NT, int R>
__device__ __forceinline__ void load_units(const Int4AttnParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v,
                                           Smem<NT>& sm, Cursor c, int64_t u0, int64_t u1, int lane) {
  int column = 0, place = 0;
  auto look_up = [&]() {
    const int pos = c.tile * kUnit + lane * 16;
    if (lane >= kParts || pos >= c.s.vis) return -1;
    const int page = ldg_keep(p.block_tables + c.seq * p.bt_stride + column);
    return page >= 0 && page < p.num_blocks ? page : -1;
  };
  auto find = [&]() {
    const int pos = c.tile * kUnit + lane * 16;
    column = pos / p.block_size;
    place = pos - column * p.block_size;
    return look_up();
  };
  int page = find();
  int stage = 0;
  uint32_t round = 0, loaded = 0;
  const bool begins = lane < kParts && lane % (p.box_rows / 16) == 0;
  bool ok = true;
  for (int64_t u = u0; u < u1; ++u) {
    const int kvh = c.pair % p.num_kv_heads;
    const int row = (page * p.num_kv_heads + kvh) * p.block_size + place;
    const bool mine = begins && page >= 0;
    const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
    const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
    // the next unit's pages
    if (u + 1 < u1) {
      if (++c.tile < c.s.tiles) {
        column += p.unit_pages;  // whole pages in a unit, and what is left
        place += p.unit_rest;
        if (place >= p.block_size) {
          place -= p.block_size;
          ++column;
        }
        page = look_up();
      } else {
        next_pair<R>(p, c);
        page = find();
      }
    }
    if (round > 0) ok = wait_warp(&sm.empty[stage], round - 1 & 1u, p.err);
    if (!ok) break;
    uint64_t* bar = &sm.full[stage];
    if (lane == 0) {
      sm.there[stage] = there;
      mbar_arrive_expect_tx(bar, boxes * p.box_rows * 136);
    }
    __syncwarp();
    if (mine) {
      tma_load_2d(sm.k[stage] + lane * 1024, &map_k, bar, 0, row);
      tma_load_2d(sm.v[stage] + lane * 1024, &map_v, bar, 0, row);
      bulk_load(smem_u32(sm.scale[stage] + lane * 16), p.kv_scale + static_cast<int64_t>(row) * 4, p.box_rows * 8, bar);
    }
    loaded |= 1u << stage;
    if (++stage == kStages) {
      stage = 0;
      ++round;
    }
  }
  // copies in flight after a wait that gave up: they must land (or run out of time) before the CTA ends
  if (!ok)
    for (int i = 0; i < kStages; ++i)
      if (loaded >> i & 1u) wait_warp(&sm.full[i], (i < stage ? round : round - 1) & 1u, p.err);
}

template <int NT, bool kFold>
__global__ void __launch_bounds__(kThreads, NT == 1 ? INT4_C : 2) int4_decode_kernel(
    const __grid_constant__ Int4AttnParams p, const __grid_constant__ CUtensorMap map_k,
    const __grid_constant__ CUtensorMap map_v) {
  extern __shared__ uint8_t smem_raw[];
  Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(smem_raw + (1024 - smem_u32(smem_raw) % 1024) % 1024);
  constexpr int R = kFold ? 4 : 8 * NT;  // rows of a group
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], kWarps);
    }
    fence_mbar_init();
  }
  // programmatic dependent of the kernel before it: nothing is read or written before that ends
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- plan: units before each sequence; thread i has sequences [i * per, (i + 1) * per)
  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += seq_of<R>(p, s).units(p.num_kv_heads);
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
  for (int w = 0; w < kWarps + 1; ++w) {
    if (w < warp) before += sm.scan[w];
    total += sm.scan[w];
  }
  before -= mine;
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);
  Cut* cuts = reinterpret_cast<Cut*>(p.cuts);
  if (blockIdx.x >= ctas) {
    if (tid == 0) cuts[blockIdx.x].parts = 0;
    return;
  }
  const int64_t u0 = range_begin(blockIdx.x, ctas, total), u1 = range_begin(blockIdx.x + 1, ctas, total);
  if (before <= u0 && u0 < before + mine) {
    int64_t at = before;
    int s = s0;
    for (; s < s1; ++s) {
      const int64_t n = seq_of<R>(p, s).units(p.num_kv_heads);
      if (u0 < at + n) break;
      at += n;
    }
    sm.first_seq = s;
    sm.first_unit = at;
  }
  __syncthreads();
  Cursor now;
  now.seq = sm.first_seq;
  now.s = seq_of<R>(p, now.seq);
  {
    const int64_t rest = u0 - sm.first_unit;
    now.pair = static_cast<int>(rest / now.s.tiles);
    now.tile = static_cast<int>(rest - static_cast<int64_t>(now.pair) * now.s.tiles);
  }

  if (warp == kWarps) {
    load_units<NT, R>(p, map_k, map_v, sm, now, u0, u1, lane);
    return;
  }

  // this lane's row for the transposed loads of V, and its piece (of the second of two: 1) as it is stored; its
  // rows g and g + 8 of K, piece t
  const int v_token = (lane & 7) + (lane & 8);
  const uint32_t v_row = (warp * kTile + v_token) * 64, v_piece = (lane >> 4) ^ (v_token >> 1 & 3);
  const uint32_t k_row = (warp * kTile + g) * 64 + (t ^ (g >> 1 & 3)) * 16;
  const uint32_t k_ring = smem_u32(sm.k[0]) + k_row, v_ring = smem_u32(sm.v[0]) + v_row;
  const uint32_t s_ring = smem_u32(sm.scale[0]) + (warp * kTile + g) * 8;
  uint32_t by8;
  asm volatile("mov.u32 %0, 0x1000000;" : "=r"(by8));
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;  // no wait has given up
  for (int64_t u = u0; u < u1;) {
    // ---- a piece: units [u, u + n) of one pair
    const int n = static_cast<int>(min(u1 - u, static_cast<int64_t>(now.s.tiles - now.tile)));
    const bool whole = now.tile == 0 && n == now.s.tiles;
    const int kvh = now.pair % p.num_kv_heads, rg = now.pair / p.num_kv_heads;
    const int rows = now.s.nq * p.group;  // of this kv head
    // q: the B operand of S^T, plane j by warp j.  Column (row) g, values 32 t .. 32 t + 31 in the order
    // of the codes
    if (warp < NT) {
      const int r = rg * R + (kFold ? g & 3 : 8 * warp + g);
      uint4 raw[4] = {};
      if (r < rows) {
        const int token = r / p.group;
        const uint16_t* src = p.q + (static_cast<int64_t>(now.s.q_first) + token) * p.q_row_stride +
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
    sync_compute();
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
        const int row = rg * R + (kFold ? (2 * t + c) & 3 : 8 * j + 2 * t + c);
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
    float m_limit[NT][2];  // m and how far it may lag
    float v_unit = 1.f, v_limit = 0.f;  // steps of V are multiplied by v_unit (a power of two)
    int v_exp = 0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[j][c] = m_limit[j][c] = kNone;
        l[j][c] = mid[j][c] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) ps[j][c] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[j][i][c] = 0.f;
    }

    for (int i = 0; i < n; ++i) {
      const int pos0 = (now.tile + i) * kUnit + warp * kTile;
      ok = ok && wait_warp(&sm.full[stage], parity, p.err);
      const uint32_t halves = sm.there[stage] >> (2 * warp) & 3u;
      if (halves != 0 && pos0 < most && ok) {
        // ---- S^T: positions (rows g, g + 8 of each half) x query rows (columns)
        float s[2][NT][4];
        uint32_t kw[2][2][4];  // half, row g or g + 8, word
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint4 k = ld_shared_v4(k_ring + stage * (kUnit * 64) + h * 1024 + r * 512);
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
              const uint32_t y0 = b ? shift8(kw[h][0][w], by8) : kw[h][0][w];
              const uint32_t y1 = b ? shift8(kw[h][1][w], by8) : kw[h][1][w];
              a[h][0] = y0 & 0x000F000Fu;
              a[h][1] = y1 & 0x000F000Fu;
              a[h][2] = y0 & 0x00F000F0u;
              a[h][3] = y1 & 0x00F000F0u;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const uint2 qb = kHeld ? q[kHeld ? j : 0][2 * w + b] : sm.q[j][2 * w + b][lane];
              if (w == 0 && b == 0) {
                mma16816_first(s[0][j], a[0], qb.x, qb.y);
                mma16816_first(s[1][j], a[1], qb.x, qb.y);
              } else {
                mma16816(s[0][j], a[0], qb.x, qb.y);
                mma16816(s[1][j], a[1], qb.x, qb.y);
              }
            }
          }
        }
        // Folded: with at most four rows the columns hold them twice, the first four go on with half 0 and the
        // last four with half 1, and the scores of a tile are half as many.
        constexpr int H = kFold ? 1 : 2;
        if constexpr (kFold) {
#pragma unroll
          for (int c = 0; c < 4; ++c) s[0][0][c] = t < 2 ? s[0][0][c] : s[1][0][c];
        }
        // ---- scores; this thread's positions: rows g and g + 8 of half h (folded: of half t >> 1)
        float sv[H][2], mv[H][2];  // step of V, and what code 7.5 stands for
        bool grow = false;
        const bool full = halves == 3u && pos0 + kTile <= least;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const int half = kFold ? t >> 1 : h;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint2 sc = ld_shared_v2(s_ring + stage * (kUnit * 8) + half * 128 + r * 64);
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
          for (int h = 0; h < H; ++h) {
            const int half = kFold ? t >> 1 : h;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int pos = pos0 + 16 * half + g + 8 * r;
              const bool held = (halves >> half & 1u) && pos < now.s.vis;
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
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            grow |= sv[h][r] > v_limit;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int c = 0; c < 2; ++c) grow |= s[h][j][2 * r + c] > m_limit[j][c];
          }
        if (__any_sync(0xffffffffu, grow)) {
          // ---- new references: the rows' maxima so far, and a power of two near V's largest step
          float top = 0.f;
#pragma unroll
          for (int h = 0; h < H; ++h) top = fmaxf(top, fmaxf(sv[h][0], sv[h][1]));
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
              float mx = m[j][c];
#pragma unroll
              for (int h = 0; h < H; ++h) mx = fmaxf(mx, fmaxf(s[h][j][c], s[h][j][2 + c]));
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              const float f = ex2(m[j][c] - mx);
              m[j][c] = mx;
              m_limit[j][c] = mx + kSlack;
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
        for (int h = 0; h < H; ++h) {
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
        if constexpr (kFold) {  // columns of the other half: nothing
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t both = pb[0][0][r];
            pb[0][0][r] = g < 4 ? both : 0u;
            pb[1][0][r] = g < 4 ? 0u : both;
          }
        }
        // ---- O^T += V^T P^T: of 32 values (a 16-byte piece) 4 g + 2 b (rows g) and 4 g + 2 b + 1 (rows g + 8,
        // codes four bits higher)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          constexpr uint32_t kOne = 0x3C003C00u;
          const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
#pragma unroll
          for (int j = 0; j < NT; ++j) mma16816(ps[j], ones, pb[h][j][0], pb[h][j][1]);
#pragma unroll
          for (int w = 0; w < 4; w += 2) {
            uint32_t v[4];  // piece w: rows 0-7 and 8-15, piece w + 1: the same
            ldmatrix_trans(v, v_ring + stage * (kUnit * 64) + h * 1024 + (w ^ v_piece) * 16);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                const uint32_t y0 = b ? shift8(v[2 * x], by8) : v[2 * x];
                const uint32_t y1 = b ? shift8(v[2 * x + 1], by8) : v[2 * x + 1];
                const uint32_t a[4] = {y0 & 0x000F000Fu, y0 & 0x00F000F0u, y1 & 0x000F000Fu, y1 & 0x00F000F0u};
#pragma unroll
                for (int j = 0; j < NT; ++j) mma16816(o[j][2 * (w + x) + b], a, pb[h][j][0], pb[h][j][1]);
              }
            }
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (lane == 0) mbar_arrive(&sm.empty[stage]);
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1u;
      }
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
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // values 32 (i >> 1) + 4 g + 2 (i & 1) and the one after it
          const float y0 = fmaf(fmaf(o[j][i][c], unit_even, -7.5f * ps[j][c]), back, mid[j][c]);
          const float y1 = fmaf(fmaf(o[j][i][2 + c], unit_odd, -7.5f * ps[j][c]), back, mid[j][c]);
          *reinterpret_cast<float2*>(&sm.o[warp][2 * t + c][32 * (i >> 1) + 4 * g + 2 * (i & 1)]) = make_float2(y0, y1);
        }
      }
      sync_compute();
      constexpr int kRows = kFold ? 4 : 8;
#pragma unroll
      for (int idx = tid; idx < kRows * 64; idx += kWarps * 32) {
        const int row = idx >> 6, value = 2 * (idx & 63);
        float mx = kNone;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          mx = fmaxf(mx, sm.m[w][row]);
          if (kFold) mx = fmaxf(mx, sm.m[w][row + 4]);
        }
        float y0 = 0.f, y1 = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
#pragma unroll
          for (int f4 = 0; f4 < (kFold ? 8 : 4); f4 += 4) {
            const float f = ex2(sm.m[w][row + f4] - mx);
            const float2 y = *reinterpret_cast<const float2*>(&sm.o[w][row + f4][value]);
            y0 = fmaf(y.x, f, y0);
            y1 = fmaf(y.y, f, y1);
            sum = fmaf(sm.l[w][row + f4], f, sum);
          }
        }
        const int in_group = 8 * j + row;
        if (whole) {
          const int r = rg * R + in_group;
          if (r < rows) {
            const int token = r / p.group;
            // 0 for a row that sees nothing
            const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
            uint16_t* dst = p.out + (static_cast<int64_t>(now.s.q_first) + token) * p.out_row_stride +
                            (kvh * p.group + r - token * p.group) * kHeadDim + value;
            *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(y0 * inv, y1 * inv);
          }
        } else {
          *reinterpret_cast<float2*>(part + in_group * kHeadDim + value) = make_float2(y0, y1);
          if (value == 0) *reinterpret_cast<float2*>(part + R * kHeadDim + 2 * in_group) = make_float2(mx, sum);
        }
      }
      sync_compute();
    }
    // ---- on to the next pair
    u += n;
    if (u < u1) {
      next_pair<R>(p, now);
    } else if (tid == 0) {
      Cut cut = {};
      if (now.tile == 0 && n < now.s.tiles) {
        cut.parts = static_cast<int>(owner(u - n + now.s.tiles - 1, ctas, total) - blockIdx.x + 1);
        cut.slot = 2 * blockIdx.x + (u - n > u0 ? 1 : 0);
        cut.rows = min(R, rows - rg * R);
        cut.first_row = rg * R;
        cut.token = now.s.q_first;
        cut.head = kvh * p.group;
      }
      cuts[blockIdx.x] = cut;
    }
  }
}

template <int NT>
constexpr int kSmemBytes = static_cast<int>(sizeof(Smem<NT>)) + 1024;  // its alignment

template <int NT, bool kFold>
cudaError_t prepare() {
  return cudaFuncSetAttribute(int4_decode_kernel<NT, kFold>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              kSmemBytes<NT>);
}

template <int NT, bool kFold>
int resident(int num_sms) {  // CTAs that run at once
  int per_sm = 0;
  if (prepare<NT, kFold>() != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, int4_decode_kernel<NT, kFold>, kThreads,
                                                    kSmemBytes<NT>) != cudaSuccess)
    return 0;
  return per_sm * num_sms;
}

template <int NT, bool kFold>
cudaError_t launch(const Int4AttnParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, int grid,
                   cudaStream_t stream) {
  cudaError_t e = prepare<NT, kFold>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes<NT>;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, int4_decode_kernel<NT, kFold>, p, map_k, map_v);
}

// The kernel for a call: 0 for at most four rows of a kv head, else planes of 8 rows in a row group, as many as the
// longest chunk's rows need, at most four.
int variant(int group, int max_q) {
  const int64_t rows = static_cast<int64_t>(group) * max_q;
  return rows <= 4 ? 0 : rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : 4;
}
int rows_of(int v) { return v == 0 ? 4 : 8 * v; }

}  // namespace

cudaError_t int4_error_word(void** word) { return cudaGetSymbolAddress(word, g_error); }

int int4_decode_grid(int group, int max_q) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> known[kMaxDevices][5];  // by device and variant; 0: not asked yet
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  const int v = variant(group, max_q);
  int n = known[dev][v].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    n = v == 0   ? resident<1, true>(sms)
        : v == 1 ? resident<1, false>(sms)
        : v == 2 ? resident<2, false>(sms)
        : v == 3 ? resident<3, false>(sms)
                 : resident<4, false>(sms);
    known[dev][v].store(n, std::memory_order_relaxed);
  }
  return n;
}

int64_t int4_decode_workspace_bytes(int group, int max_q, int grid) {
  const int64_t part = static_cast<int64_t>(rows_of(variant(group, max_q))) * (kHeadDim + 2) * 4;
  return static_cast<int64_t>(grid) * (kInt4CutBytes + 2 * part);
}

int int4_decode_rows(int group, int max_q) { return rows_of(variant(group, max_q)); }

cudaError_t launch_int4_decode(Int4AttnParams p, const CUtensorMap& map_k, const CUtensorMap& map_v, int grid,
                               cudaStream_t stream) {
  p.unit_pages = kUnit / p.block_size;
  p.unit_rest = kUnit % p.block_size;
  switch (variant(p.group, p.max_q)) {
    case 0: return launch<1, true>(p, map_k, map_v, grid, stream);
    case 1: return launch<1, false>(p, map_k, map_v, grid, stream);
    case 2: return launch<2, false>(p, map_k, map_v, grid, stream);
    case 3: return launch<3, false>(p, map_k, map_v, grid, stream);
    default: return launch<4, false>(p, map_k, map_v, grid, stream);
  }
}

}  // namespace fp8attn
