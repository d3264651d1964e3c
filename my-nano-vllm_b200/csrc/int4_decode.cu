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
// Bound by HBM up to 8 rows: 136 bytes of K and V for each position and kv head, read once for all of the rows of
// its query heads (64 sequences of 32,768, 8 rows: 405 us, 0.86 of the floor at 6.55 TB/s; 4 rows: 399 us).  Above,
// by the tensor cores of mma.sync: 34 products of 8 cycles for each 32 positions and plane of 8 rows, which fp32
// arithmetic does not overlap (8 fma beside one product: 14.9 cycles, and 8 without it), against 186 cycles of
// HBM: 16 rows 587 us, 24 rows 779, 32 rows 1,059.
//
// Work: a unit is 128 positions of one (sequence, row group, kv head), and a warp computes S^T = K q^T and P of 32 of
// them (A = codes, 16 positions x 16 values).  P goes through shared memory (stmatrix turns it), and of all 128
// positions the warp adds O^T += V^T P^T for its 32 values (A = codes again, turned by ldmatrix).  So a warp's sums are
// 8 registers for 8 rows and not 32, and no sums are added at the end.  (Measured when 8 rows took 382 us and 24 rows 720: with
// all values in one warp 410 and 800, with q in registers instead of shared memory, which spills, 24 rows 845.)
//
// All units in order are cut into equal ranges, one for each resident CTA, wherever the cuts fall: no counters, no
// order that depends on timing.  A CTA's first and last piece may be parts of a pair; their sums go to the workspace,
// and a second kernel joins the parts of each cut pair in order.  One warp loads (TMA, 64B swizzle), three units ahead
// and across the ends of pieces.
//
// c - 7.5 is the product with c and 7.5 times the same product with ones: taken about the middle of the codes, the
// roundings of P and the cuts of the tensor cores' sums (2^-24 of each partial sum, all one way) are in proportion to
// the values and not to their distance from the row's lowest one.  A warp takes the ones of its own 32 positions, so
// their cuts are not those of the other products and do not cancel them; every 8 units (16 for more than 16 rows) the sums
// so far are put aside and later added with rounding to nearest, so that the cuts stay those of 64 instructions and do
// not grow with the context.  Off in the 2-norm, of which the output's own rounding is 1.66e-3: decode of 32,768 positions
// 1.70e-3, of 131,072 1.84e-3 (every 64 units: 1.86e-3 and 2.05e-3, 2.5 % faster; every 16: 1.72e-3 and 1.95e-3, 1 %
// faster).  The ones of all positions in one warp cancel more (every 32 units 1.70e-3 and 1.83e-3), but decode takes 4 %
// longer and verification 9 %.
//
// Precision: scores, statistics and sums in fp32; P step is rounded once, to f16 (2^-12), after its row's
// reference maximum and a power of two near the largest step of V so far are taken out, so it stays below 2^15.  That power
// is the CTA's, and so comes from rows as well that a query row does not look at.  Where steps of V differ by more than
// some 2^15 (or are zero beside others), or values pass 2^90, the rest of the piece is done with a power for each query row
// instead, that of its own largest p |v| so far, found with an exchange of maxima in every unit; what a row gets is then as
// exact as its own largest terms (64 sequences of 32,768: 405 us, 541 with one row in 64 of 2^-24).  The units of such
// pieces have a loop of their own: as a branch of the other one 24 rows took 3 % longer and 32 rows 4 % (spills).
#include <atomic>
#include <climits>
#include <type_traits>

#include "int4_attention.cuh"

namespace fp8attn {
namespace {

// The error word of these kernels' launches: it lives as long as the library's module, so that captured graphs may
// hold its address.
__device__ int g_error = 0;

constexpr int kTile = 32;               // positions of a unit whose scores a warp computes
constexpr float kSlack = 8.f;           // a reference maximum may lag by 2^8
constexpr int kStepBits = 3;            // V's largest step is 2^3 .. 2^4 when it is new, and may grow to 2^7: P step < 2^15
constexpr int kSpreadBits = 15;          // and the smallest 2^-15 of what the largest was when it was new: P step of p = 1 is 2^-12
                                        // or more there, f16's absolute error of 2^-25 relative 2^-13
constexpr float kHuge = 0x1p90f;        // sums over the positions of larger values could pass fp32's range
constexpr int kOwnBits = 14;            // of a query row's own power: P step < 2^13
constexpr int kPieceUnits = 1;          // what a pair costs beside its tiles, in units of a tile

constexpr int kWarps = 4;                    // that compute; one more loads
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kUnit = kTile * kWarps;        // positions per unit
constexpr int kParts = kUnit / 16;           // parts of a unit that lie in one page each

// A kernel by the rows of a group: NT planes of 8.  As many CTAs on an SM as have room for their sums without spilling
// (verification with 20 rows: three CTAs of 128 registers and two stages 242 us, two of 168 with three 222; 64 sequences of
// 32,768 with 32 rows: 1,413 and 1,090 us).  kFlush: units whose products with V the tensor cores add up; more
// registers take longer to be put aside (24 rows at 32,768 positions, every 8 units: 800 us and 1.70e-3 off, every 16: 780
// and 1.72e-3).
template <int NT_>
struct Shape {
  static constexpr int NT = NT_;
  static constexpr int R = 8 * NT;
  static constexpr int kCtas = NT < 3 ? 3 : 2;    // on an SM
  static constexpr int kStages = 3;
  static constexpr int kFlush = NT < 3 ? 8 : 16;
};

constexpr int kPPitch = kUnit + 8;  // bank spread

template <typename S>
struct __align__(1024) Smem {
  uint8_t k[S::kStages][kUnit * 64];  // TMA tiles of 64-byte rows, 64B swizzle: bits 1 and 2 of a row's number
  uint8_t v[S::kStages][kUnit * 64];  // change the place of its 16-byte pieces
  uint2 scale[S::kStages][kUnit];
  uint16_t rows[S::R][kHeadDim];            // q of a piece
  uint2 q[S::NT][8][32];                    // as the B operand of S^T: plane, step, lane
  uint16_t p[2][S::R][kPPitch];             // P step, f16, of this unit and the one before
  float kq[S::R], qs[S::R];                 // score = dot kq step + qs low
  float top[kWarps][S::R], term[kWarps][S::R];  // of the warps' positions: largest score and term,
  float top_v[kWarps], least_v[kWarps];  // largest and smallest step (-1: huge values),
  float l[kWarps][S::R], mid[kWarps][S::R], ps[kWarps][S::R];  // sums
  uint64_t full[S::kStages], empty[S::kStages], q_full, q_free;
  uint32_t there[S::kStages];  // which parts of the stage's unit are in pages of the cache
  int scan[kThreads / 32];
  int first_seq, first_unit;   // the sequence in which the CTA's range begins, its first unit
};

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

__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
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

__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// Four 8 x 8 matrices stored transposed: lanes 8 i .. 8 i + 7 give the rows of matrix i in shared memory.
__device__ __forceinline__ void stmatrix_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

// A barrier of the computing warps: whether x holds in any thread.
__device__ __forceinline__ bool any_warp(bool x) {
  uint32_t any;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.or.pred q, 1, %2, p;\nselp.u32 %0, 1, 0, q;\n}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(x)), "n"(kWarps * 32)
      : "memory");
  return any != 0;
}

// A sequence's rows and visible positions; units in all.
struct Seq {
  int q_first, nq, nk, vis, tiles, groups;
  __device__ __forceinline__ int units(int kvh) const { return (tiles + kPieceUnits) * groups * kvh; }  // launch: < 2^31
};

template <typename S>
__device__ __forceinline__ Seq seq_of(const Int4AttnParams& p, int s) {
  Seq q;
  if (p.cu_q != nullptr) {
    q.q_first = __ldg(p.cu_q + s);
    q.nq = __ldg(p.cu_q + s + 1) - q.q_first;
    q.nk = __ldg(p.cu_k + s + 1) - __ldg(p.cu_k + s);
    if (q.nq > p.max_q) q.nq = 0;  // the other kernel's
  } else {
    q.q_first = s;
    q.nq = 1;
    q.nk = __ldg(p.context_lens + s);
  }
  q.vis = max(0, min(q.nk, p.max_blocks * p.block_size));
  // a sequence without positions still has its zeros written
  q.tiles = max(1, (q.vis + kUnit - 1) / kUnit);
  q.groups = q.nq <= 0 ? 0 : (q.nq * p.group + S::R - 1) / S::R;
  return q;
}

// The token of a kv head's row r, of nq group < 2^31 / group
__device__ __forceinline__ int token_of(const Int4AttnParams& p, int r) { return __umulhi(2 * r, p.group_inverse); }

// The piece that a warp is at: tiles [tile, end) of a pair (row group, kv head).  A pair's units are kPieceUnits for what
// it costs beside its tiles, and then its tiles; a piece is what of it lies in the CTA's range, which ends at unit `until`.
struct Cursor {
  int seq, rg, kvh, tile, end;
  int begin, until;  // the pair's first unit
  Seq s;
  // Whether another piece with a tile follows.
  __device__ __forceinline__ bool more() const { return begin + s.tiles + 2 * kPieceUnits < until; }
  __device__ __forceinline__ void set_end() {
    end = max(0, min(s.tiles, until - begin - kPieceUnits));
  }
};

template <typename S>
__device__ __forceinline__ void next_piece(const Int4AttnParams& p, Cursor& c) {
  c.tile = 0;
  c.begin += c.s.tiles + kPieceUnits;
  if (++c.kvh >= p.num_kv_heads) {
    c.kvh = 0;
    if (++c.rg >= c.s.groups) {
      c.rg = 0;
      do {  // there is one: more()
        c.s = seq_of<S>(p, ++c.seq);
      } while (c.s.groups == 0);
    }
  }
  c.set_end();
}

// A row of q as lanes 4 g .. 4 g + 3 hold it for column g of the B operand of S^T: values 32 t .. 32 t + 31 in the order
// of the codes.  A power of two puts the row's largest value between 2^13 and 2^14; odd values, whose codes stand four
// bits higher, / 16.
__device__ __forceinline__ void convert_q(const uint16_t* row, bool is_row, int t, float scale_log2, uint2 (&q)[8],
                                          float& kq, float& qs) {
  uint4 raw[4] = {};
  if (is_row) {
#pragma unroll
    for (int w = 0; w < 4; ++w) raw[w] = *reinterpret_cast<const uint4*>(row + 32 * t + 8 * w);
  }
  float amax = 0.f, sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t word[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x0 = __uint_as_float(word[i] << 16), x1 = __uint_as_float(word[i] & 0xFFFF0000u);
      amax = fmaxf(amax, fmaxf(fabsf(x0), fabsf(x1)));
      sum += x0 + x1;
    }
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    sum += __shfl_xor_sync(0xffffffffu, sum, off);
  }
  const int e = amax > 0.f && amax < INFINITY ? max(-113, exponent(amax)) - 13 : 0;
  const float even = pow2(-e), odd = pow2(-e - 4);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t word[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
    for (int b = 0; b < 2; ++b) {  // values 2 b and 2 b + 4; 2 b + 1 and 2 b + 5
      const uint32_t lo = word[b], hi = word[b + 2];
      q[2 * w + b] = make_uint2(pack_f16x2(__uint_as_float(lo << 16) * even, __uint_as_float(hi << 16) * even),
                                pack_f16x2(__uint_as_float(lo & 0xFFFF0000u) * odd,
                                           __uint_as_float(hi & 0xFFFF0000u) * odd));
    }
  }
  kq = pow2(e) * scale_log2 * 16777216.f;  // inside fp32 up to q = 2^116 / scale
  qs = sum * scale_log2;
}

// Loads by one warp: a piece's rows of q (lane i: row i), and its units: lane i looks up the page of part i, and the
// lanes at which a TMA box of box_rows positions begins load K, V and scales.
template <typename S>
__device__ __forceinline__ void load(const Int4AttnParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v,
                                     Smem<S>& sm, Cursor c, int lane) {
  int column = 0, place = 0, page = -1, stage = 0;
  uint32_t round = 0, loaded = 0, pieces = 0;
  const bool begins = lane < kParts && lane % (p.box_rows / 16) == 0;
  bool ok = true, first = true;  // the unit is its piece's first
  auto look_up = [&]() {
    const int pos = c.tile * kUnit + lane * 16;
    page = -1;
    if (lane < kParts && pos < c.s.vis) {
      const int found = ldg_keep(p.block_tables + c.seq * p.bt_stride + column);
      if (found >= 0 && found < p.num_blocks) page = found;
    }
  };
  auto find = [&]() {
    const int pos = c.tile * kUnit + lane * 16;
    column = pos / p.block_size;
    place = pos - column * p.block_size;
    look_up();
  };
  find();
#pragma unroll 1
  for (;;) {
    if (first) {
      const int rows = c.s.nq * p.group - c.rg * S::R;  // from the group's first on
      if (pieces > 0) ok = wait_all(&sm.q_free, (pieces - 1) & 1u, p.err);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&sm.q_full, min(S::R, rows) * kHeadDim * 2);
      __syncwarp();
      if (lane < S::R && lane < rows) {
        const int r = c.rg * S::R + lane, token = token_of(p, r);
        bulk_load(smem_u32(sm.rows[lane]),
                  p.q + (static_cast<int64_t>(c.s.q_first) + token) * p.q_row_stride +
                      (c.kvh * p.group + r - token * p.group) * kHeadDim,
                  kHeadDim * 2, &sm.q_full);
      }
      ++pieces;
      first = false;
    }
    const int row = (page * p.num_kv_heads + c.kvh) * p.block_size + place;
    const bool mine = begins && page >= 0;
    const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
    const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
    // the next unit's pages
    bool more = true;
    if (++c.tile < c.end) {
      column += p.unit_pages;  // whole pages in a unit, and what is left
      place += p.unit_rest;
      if (place >= p.block_size) {
        place -= p.block_size;
        ++column;
      }
      look_up();
    } else if (c.more()) {
      next_piece<S>(p, c);
      find();
      first = true;
    } else {
      more = false;
    }
    if (round > 0) ok = wait_all(&sm.empty[stage], (round - 1) & 1u, p.err);
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
    if (++stage == S::kStages) {
      stage = 0;
      ++round;
    }
    if (!more) return;
  }
  // a wait gave up: the copies in flight must land (or run out of time) before the CTA ends
  for (int i = 0; i < S::kStages; ++i)
    if (loaded >> i & 1u) wait_all(&sm.full[i], (i < stage ? round : round - 1) & 1u, p.err);
  if (pieces > 0) wait_all(&sm.q_full, (pieces - 1) & 1u, p.err);
}

// The pair that the CTA's range leaves cut, if its last piece is one's beginning: for the joining kernel.
template <typename S>
__device__ __forceinline__ void store_cut(const Int4AttnParams& p, const Cursor& now, const Ranges& ranges,
                                          uint32_t pieces) {
  Cut cut = {};
  if (now.tile == 0 && now.end < now.s.tiles) {
    const int first = now.begin + kPieceUnits, last = first + now.s.tiles - 1;  // its tiles, as units
    cut.parts = ranges.owner(last) - ranges.owner(first) + 1;
    cut.slot = 2 * blockIdx.x + (pieces > 0 ? 1 : 0);
    cut.rows = min(S::R, now.s.nq * p.group - now.rg * S::R);
    cut.first_row = now.rg * S::R;
    cut.token = now.s.q_first;
    cut.head = now.kvh * p.group;
  }
  reinterpret_cast<Cut*>(p.cuts)[blockIdx.x] = cut;
}

// Scores, softmax and sums by four warps, which meet once for each unit: whether one of them needs new reference
// maxima, and with it, that P is there.
template <typename S>
__device__ __forceinline__ void compute(const Int4AttnParams& p, Smem<S>& sm, Cursor now, const Ranges& ranges, int warp,
                                        int lane) {
  constexpr int NT = S::NT, R = S::R;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t k_ring = smem_u32(sm.k[0]) + (warp * kTile + g) * 64 + (t ^ (g >> 1 & 3)) * 16;
  const uint32_t v_ring = smem_u32(sm.v[0]) + lane * 64 + (warp ^ (lane >> 1 & 3)) * 16;
  const uint32_t s_ring = smem_u32(sm.scale[0]) + (warp * kTile + g) * 8;
  const uint32_t s_own = s_ring + (t >> 1) * 128 + (t & 1) * 64 + 4;
  const uint32_t p_lane = smem_u32(sm.p[0]) + ((lane & 7) * kPPitch + (lane >> 3) * 8) * 2;  // row of a plane, 8 positions
  auto all_warps = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); };
  int stage = 0;
  uint32_t parity = 0, pieces = 0, p_buf = 0;
  bool ok = true;  // no wait has given up
#pragma unroll 1
  for (;; ++pieces) {
    const int n = now.end - now.tile, kvh = now.kvh, rg = now.rg;
    const int rows = now.s.nq * p.group;  // of this kv head
    ok = ok && wait_all(&sm.q_full, pieces & 1u, p.err);
    if (warp < NT) {
      uint2 y[8];
      float a, b;
      convert_q(sm.rows[8 * warp + g], rg * R + 8 * warp + g < rows, t, p.scale_log2, y, a, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) sm.q[warp][i][lane] = y[i];
      if (t == 0) {
        sm.kq[8 * warp + g] = a;
        sm.qs[8 * warp + g] = b;
      }
    }
    all_warps();
    if (lane == 0) mbar_arrive(&sm.q_free);
    auto limit_of = [&](int j, int c) {  // positions that a column's row sees; where there is no row, as the group's first
      int row = rg * R + 8 * j + 2 * t + c;
      if (row >= rows) row = rg * R;
      return min(now.s.vis, token_of(p, row) + now.s.nk - now.s.nq + 1);
    };
    int least = INT_MAX;
#pragma unroll
    for (int j = 0; j < NT; ++j) least = min(least, min(limit_of(j, 0), limit_of(j, 1)));
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, off));

    float o[NT][2][4], ps[NT][4];          // ps: sum of the rounded P step, of this warp's positions
    // in local memory: o and ps of the units before, their m and power; columns' own powers (`own`)
    volatile float kept[10 * NT], m_kept[2 * NT], power_kept[2 * NT], power[2 * NT];
    uint64_t minus_m[NT], l[NT], mid[NT];  // pairs of columns
    uint32_t unset = (1u << 2 * NT) - 1;   // columns that have seen nothing: their m counts as 0
    float limit = -INFINITY;               // how far a score may be above its m: kSlack when none is unset
    float v_unit = 1.f, v_limit = 0.f;     // steps of V are multiplied by v_unit (a power of two)
    float v_floor = 0.f, v_least = 3.402823466e38f;  // steps are to be v_floor or more; the smallest so far
    int v_exp = 0;
    bool own = false;                      // columns have powers of their own: o is in units of 2^(power - kOwnBits), mid of 2^power
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      minus_m[j] = l[j] = mid[j] = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) ps[j][c] = o[j][0][c] = o[j][1][c] = 0.f;
    }
    auto unit_of = [&](int column) { return own ? power[column] - kOwnBits : static_cast<float>(v_exp); };
    auto add_kept = [&]() {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float m[2];
        f2_unpack(minus_m[j], m[0], m[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float f = ex2((m[c] - m_kept[2 * j + c]) + (power_kept[2 * j + c] - unit_of(2 * j + c)));
          auto add = [&](float& x, float y) { x += y == 0.f ? 0.f : y * f; };  // 0 where nothing had been seen
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            add(o[j][b][c], kept[8 * j + 4 * b + c]);
            add(o[j][b][2 + c], kept[8 * j + 4 * b + 2 + c]);
          }
          add(ps[j][c], kept[8 * NT + 2 * j + c]);
        }
      }
    };
    // Unit i of the piece.  False (and nothing done): its rows of V need columns' own powers, as they have with kOwn.
    auto unit = [&](const int i, auto with_own) -> bool {
      constexpr bool kOwn = decltype(with_own)::value;
      const int pos0 = (now.tile + i) * kUnit + warp * kTile;
      ok = ok && wait_all(&sm.full[stage], parity, p.err);
      const uint32_t halves = sm.there[stage] >> (2 * warp) & 3u;
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
            const uint32_t y0 = kw[h][0][w] >> (8 * b);
            const uint32_t y1 = kw[h][1][w] >> (8 * b);
            a[h][0] = y0 & 0x000F000Fu;
            a[h][1] = y1 & 0x000F000Fu;
            a[h][2] = y0 & 0x00F000F0u;
            a[h][3] = y1 & 0x00F000F0u;
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint2 y = sm.q[j][2 * w + b][lane];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (w == 0 && b == 0) mma16816_first(s[h][j], a[h], y.x, y.y);
              else mma16816(s[h][j], a[h], y.x, y.y);
            }
          }
        }
      }
      // ---- scores above their m; this thread's positions: rows g and g + 8 of half h
      float sv[2][2], mv[2][2];  // step of V, and what code 7.5 stands for
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint2 sc = ld_shared_v2(s_ring + stage * (kUnit * 8) + h * 128 + r * 64);
          const float sk = __uint_as_float(sc.x << 16), lk = __uint_as_float(sc.x & 0xFFFF0000u);
          sv[h][r] = __uint_as_float(sc.y << 16);
          mv[h][r] = fmaf(7.5f, sv[h][r], __uint_as_float(sc.y & 0xFFFF0000u));
          const uint64_t sk2 = f2_pack(sk, sk), lk2 = f2_pack(lk, lk);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint64_t kq = reinterpret_cast<const uint64_t*>(sm.kq)[4 * j + t];
            const uint64_t qs = reinterpret_cast<const uint64_t*>(sm.qs)[4 * j + t];
            const uint64_t x = f2_fma(f2_pack(s[h][j][2 * r], s[h][j][2 * r + 1]), f2_mul(sk2, kq),
                                      f2_fma(lk2, qs, minus_m[j]));
            f2_unpack(x, s[h][j][2 * r], s[h][j][2 * r + 1]);
          }
        }
      }
      // of the four threads that have the same positions, each looks after one: V's step and lowest value
      float step, low;
      {
        const uint32_t sc = ld_shared_u32(s_own + stage * (kUnit * 8));
        step = __uint_as_float(sc << 16);
        low = __uint_as_float(sc & 0xFFFF0000u);
      }
      if (halves != 3u || pos0 + kTile > least) {
        int sees[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          sees[j][0] = limit_of(j, 0);
          sees[j][1] = limit_of(j, 1);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int pos = pos0 + 16 * h + g + 8 * r;
            const bool held = (halves >> h & 1u) && pos < now.s.vis;
            // a row of V that is no number goes to those that see it by their scores
            const bool number = fabsf(mv[h][r]) < INFINITY;
            if (!held || !number) {
              sv[h][r] = mv[h][r] = 0.f;
              if (t == 2 * h + r) step = low = NAN;  // neither large nor small
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                if (!number) s[h][j][2 * r + c] = NAN;
                if (!held || pos >= sees[j][c]) s[h][j][2 * r + c] = -INFINITY;
              }
            }
          }
        }
      }
      const uint32_t p_at = p_lane + p_buf * (R * kPPitch * 2);
      uint64_t l_now[NT], mid_now[NT];
      if constexpr (!kOwn) {
        v_least = fminf(v_least, step);
        bool grow = step > v_limit || v_least < v_floor || fabsf(low) > kHuge;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
            grow |= fmaxf(fmaxf(s[h][j][0], s[h][j][1]), fmaxf(s[h][j][2], s[h][j][3])) > limit;
        }
        // ---- P, and P step_v to shared memory: [row][position]
        auto give_p = [&]() {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            uint32_t x[2][2];
            l_now[j] = l[j];
            mid_now[j] = mid[j];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const uint64_t e = f2_pack(ex2(s[h][j][2 * r]), ex2(s[h][j][2 * r + 1]));
                const float f = sv[h][r] * v_unit;
                l_now[j] = f2_add(l_now[j], e);
                mid_now[j] = f2_fma(e, f2_pack(mv[h][r], mv[h][r]), mid_now[j]);
                float p0, p1;
                f2_unpack(f2_mul(e, f2_pack(f, f)), p0, p1);
                x[h][r] = pack_f16x2(p0, p1);
              }
            }
            stmatrix_trans(p_at + (8 * j * kPPitch + warp * kTile) * 2, x[0][0], x[0][1], x[1][0], x[1][1]);
          }
        };
        give_p();
        if (any_warp(grow)) {
          // ---- new references, of the CTA: the rows' maxima so far, and a power of two near V's largest step
          float top = fmaxf(step, 0.f);
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const uint32_t small = __reduce_min_sync(0xffffffffu, __float_as_uint(v_least));  // none is negative
          const bool big = __any_sync(0xffffffffu, fabsf(low) > kHuge || step > kHuge);
          if (lane == 0) {
            sm.top_v[warp] = top;
            sm.least_v[warp] = big ? -1.f : __uint_as_float(small);
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = fmaxf(fmaxf(s[0][j][c], s[0][j][2 + c]), fmaxf(s[1][j][c], s[1][j][2 + c]));
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              if (g == 0) sm.top[warp][8 * j + 2 * t + c] = mx;
            }
          }
          all_warps();
          float change = 1.f, smallest = sm.least_v[0];
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            top = fmaxf(top, sm.top_v[w]);
            smallest = fminf(smallest, sm.least_v[w]);
          }
          const bool larger = top > v_limit && top < INFINITY;
          const int x = max(-120, min(exponent(top), 120));
          if (larger) v_floor = pow2(max(x - kSpreadBits, -126));
          if (smallest < v_floor) return false;
          if (larger) {
            if (v_limit > 0.f) {
              const int d = v_exp - (x - kStepBits);
              change = d < -126 ? 0.f : pow2(d);
            }
            v_exp = x - kStepBits;
            v_unit = pow2(-v_exp);
            v_limit = pow2(x + 4);
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float was[2], now_m[2], f[2];
            f2_unpack(minus_m[j], was[0], was[1]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = -INFINITY;  // above m
#pragma unroll
              for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm.top[w][8 * j + 2 * t + c]);
              const bool first = unset >> (2 * j + c) & 1u;
              if (first && mx == -INFINITY) mx = 0.f;  // still unset
              else unset &= ~(1u << (2 * j + c));
              if (!first) mx = fmaxf(mx, 0.f);
              f[c] = first ? 0.f : ex2(-mx);
              now_m[c] = was[c] - mx;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                s[h][j][c] -= mx;
                s[h][j][2 + c] -= mx;
              }
              ps[j][c] *= f[c] * change;
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                o[j][b][c] *= f[c] * change;
                o[j][b][2 + c] *= f[c] * change;
              }
            }
            minus_m[j] = f2_pack(now_m[0], now_m[1]);
            l[j] = f2_mul(l[j], f2_pack(f[0], f[1]));
            mid[j] = f2_mul(mid[j], f2_pack(f[0], f[1]));
          }
          limit = __any_sync(0xffffffffu, unset != 0) ? -INFINITY : kSlack;
          give_p();
          all_warps();
        }
      } else {
        // ---- rows' maxima, and their largest terms (of the units before the first of these: their sums), each time anew
        float ex[2][2];  // exponents of V's rows
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            ex[h][r] = static_cast<float>(max(-126, min(exponent(fmaf(7.5f, sv[h][r], fabsf(mv[h][r]))), 126)));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float middle[2];
          f2_unpack(mid[j], middle[0], middle[1]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            auto power_of = [](float x, int e) { return x == 0.f ? -1000.f : static_cast<float>(exponent(fabsf(x)) + e); };
            float term = own ? power[2 * j + c] : fmaxf(power_of(middle[c], 1), power_of(ps[j][c], v_exp + 4));
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              mx = fmaxf(mx, fmaxf(s[h][j][c], s[h][j][2 + c]));
              term = fmaxf(term, fmaxf(s[h][j][c] + ex[h][0], s[h][j][2 + c] + ex[h][1]));
            }
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              term = fmaxf(term, __shfl_xor_sync(0xffffffffu, term, off));
            }
            if (g == 0) {
              sm.top[warp][8 * j + 2 * t + c] = mx;
              sm.term[warp][8 * j + 2 * t + c] = term;
            }
          }
        }
        all_warps();
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float was[2], now_m[2], f[2], mid_to[2], to[2];
          f2_unpack(minus_m[j], was[0], was[1]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int column = 8 * j + 2 * t + c;
            float mx = -INFINITY, term = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              mx = fmaxf(mx, sm.top[w][column]);
              term = fmaxf(term, sm.term[w][column]);
            }
            const bool first = unset >> (2 * j + c) & 1u;
            if (first && mx == -INFINITY) mx = 0.f;
            else unset &= ~(1u << (2 * j + c));
            if (!first) mx = fmaxf(mx, 0.f);
            f[c] = first ? 0.f : ex2(-mx);
            now_m[c] = was[c] - mx;
            to[c] = fmaxf(ceilf(term - mx), -200.f);
            // sums of nothing may be multiplied by anything
            const float o_to = ex2(fminf((own ? power[2 * j + c] : static_cast<float>(v_exp + kOwnBits)) - mx - to[c], 100.f));
            mid_to[c] = ex2(fminf((own ? power[2 * j + c] : 0.f) - mx - to[c], 100.f));
            power[2 * j + c] = to[c];
            ps[j][c] *= o_to;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              o[j][b][c] *= o_to;
              o[j][b][2 + c] *= o_to;
            }
          }
          minus_m[j] = f2_pack(now_m[0], now_m[1]);
          l_now[j] = f2_mul(l[j], f2_pack(f[0], f[1]));
          mid_now[j] = f2_mul(mid[j], f2_pack(mid_to[0], mid_to[1]));
          // ---- P: V's row by its own power, and that power beside the score's
          uint32_t x[2][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float down = pow2(-static_cast<int>(ex[h][r])), step = sv[h][r] * down * static_cast<float>(1 << kOwnBits);
              const float s0 = s[h][j][2 * r] + (now_m[0] - was[0]), s1 = s[h][j][2 * r + 1] + (now_m[1] - was[1]);
              const uint64_t e = f2_pack(ex2(s0 + (ex[h][r] - to[0])), ex2(s1 + (ex[h][r] - to[1])));
              float p0, p1;
              l_now[j] = f2_add(l_now[j], f2_pack(ex2(s0), ex2(s1)));
              mid_now[j] = f2_fma(e, f2_pack(mv[h][r] * down, mv[h][r] * down), mid_now[j]);
              f2_unpack(f2_mul(e, f2_pack(step, step)), p0, p1);
              x[h][r] = pack_f16x2(p0, p1);
            }
          }
          stmatrix_trans(p_at + (8 * j * kPPitch + warp * kTile) * 2, x[0][0], x[0][1], x[1][0], x[1][1]);
        }
        own = true;
        all_warps();
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        l[j] = l_now[j];
        mid[j] = mid_now[j];
      }
      // ---- sums of P step_v: of this warp's positions
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        constexpr uint32_t kOne = 0x3C003C00u;
        const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
        uint32_t b[4];
        ldmatrix(b, p_at + (8 * j * kPPitch + warp * kTile) * 2);
        mma16816(ps[j], ones, b[0], b[1]);
        mma16816(ps[j], ones, b[2], b[3]);
      }
      // ---- O^T += V^T P^T: of its 32 values 4 g + 2 b (rows g) and 4 g + 2 b + 1 (rows g + 8, codes four bits higher)
#pragma unroll
      for (int x = 0; x < kUnit / 32; ++x) {
        uint32_t v[4], pb[NT][4];  // of 8 positions each
        ldmatrix_trans(v, v_ring + stage * (kUnit * 64) + x * 2048);
#pragma unroll
        for (int j = 0; j < NT; ++j) ldmatrix(pb[j], p_at + (8 * j * kPPitch + x * 32) * 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint32_t y0 = v[2 * h] >> (8 * b), y1 = v[2 * h + 1] >> (8 * b);
            const uint32_t a[4] = {y0 & 0x000F000Fu, y0 & 0x00F000F0u, y1 & 0x000F000Fu, y1 & 0x00F000F0u};
#pragma unroll
            for (int j = 0; j < NT; ++j) mma16816(o[j][b], a, pb[j][2 * h], pb[j][2 * h + 1]);
          }
        }
      }
      p_buf ^= 1u;
      __syncwarp();  // every lane has read the stage
      if (lane == 0) mbar_arrive(&sm.empty[stage]);
      if (++stage == S::kStages) {
        stage = 0;
        parity ^= 1u;
      }
      return true;
    };
#pragma unroll 1
    for (int i = 0; i < n;) {
      const int stop = min(n, (i / S::kFlush + 1) * S::kFlush);
      if (!own) {
#pragma unroll 1
        for (; i < stop; ++i)
          if (!unit(i, std::false_type())) break;
      }
#pragma unroll 1
      for (; i < stop; ++i) unit(i, std::true_type());
      // ---- the sums so far, rounded to nearest: the tensor cores' cuts, all one way, stay those of so many
      if (i > S::kFlush) add_kept();
      if (i < n) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float m[2];
          f2_unpack(minus_m[j], m[0], m[1]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            m_kept[2 * j + c] = m[c];
            power_kept[2 * j + c] = unit_of(2 * j + c);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            kept[8 * j + c] = o[j][0][c];
            kept[8 * j + 4 + c] = o[j][1][c];
            if (c < 2) kept[8 * NT + 2 * j + c] = ps[j][c];
            ps[j][c] = o[j][0][c] = o[j][1][c] = 0.f;
          }
        }
      }
    }

    // ---- the rows' sums over the warps' positions, and outputs of a whole pair or a part for the joining kernel
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float sum[2], middle[2];
      f2_unpack(l[j], sum[0], sum[1]);
      f2_unpack(mid[j], middle[0], middle[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], off);
          middle[c] += __shfl_xor_sync(0xffffffffu, middle[c], off);
        }
        if (g == 0) {
          sm.l[warp][8 * j + 2 * t + c] = sum[c];
          sm.mid[warp][8 * j + 2 * t + c] = middle[c];
          sm.ps[warp][8 * j + 2 * t + c] = ps[j][c];
        }
      }
    }
    all_warps();
    const bool whole = now.tile == 0 && now.end == now.s.tiles;
    const float unit_even = 16777216.f, unit_odd = 1048576.f, back = own ? 1.f / (1 << kOwnBits) : pow2(v_exp);
    float* const part = p.partials + static_cast<int64_t>(2 * blockIdx.x + (pieces > 0 ? 1 : 0)) * (R * (kHeadDim + 2));
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float m[2];
      f2_unpack(minus_m[j], m[0], m[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int column = 8 * j + 2 * t + c, r = rg * R + column;
        float sum = 0.f, middle = 0.f, steps = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          sum += sm.l[w][column];
          middle += sm.mid[w][column];
          steps += sm.ps[w][column];
        }
        float y[4];  // values 4 g .. 4 g + 3 of the warp's
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          y[2 * b] = fmaf(fmaf(o[j][b][c], unit_even, -7.5f * steps), back, middle);
          y[2 * b + 1] = fmaf(fmaf(o[j][b][2 + c], unit_odd, -7.5f * steps), back, middle);
        }
        if (r >= rows || !ok) continue;
        const int value = 32 * warp + 4 * g;
        const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);  // 0 for a row that sees nothing
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] *= inv;
        if (own) {  // in two steps: the power may be beyond fp32's
          const int e = static_cast<int>(power[2 * j + c]), e0 = e / 2;
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = y[k] * pow2(e0) * pow2(e - e0);
        }
        if (whole) {
          const int token = token_of(p, r);
          const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]);
          const __nv_bfloat162 hi = __floats2bfloat162_rn(y[2], y[3]);
          *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(now.s.q_first) + token) * p.out_row_stride +
                                    (kvh * p.group + r - token * p.group) * kHeadDim + value) =
              make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        } else {
          *reinterpret_cast<float4*>(part + column * kHeadDim + value) = make_float4(y[0], y[1], y[2], y[3]);
          if (warp == 0 && g == 0)
            *reinterpret_cast<float2*>(part + R * kHeadDim + 2 * column) =
                make_float2(unset >> (2 * j + c) & 1u ? kNone : -m[c], sum);
        }
      }
    }
    // ---- on to the next pair
    if (!now.more()) {
      if (warp == 0 && lane == 0) store_cut<S>(p, now, ranges, pieces);
      return;
    }
    next_piece<S>(p, now);
  }
}

template <typename S>
__global__ void __launch_bounds__(kThreads, S::kCtas)
    int4_decode_kernel(const __grid_constant__ Int4AttnParams p, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v) {
  extern __shared__ uint8_t smem_raw[];
  Smem<S>& sm = *reinterpret_cast<Smem<S>*>(smem_raw + (1024 - smem_u32(smem_raw) % 1024) % 1024);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], kWarps);
    }
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_free, kWarps);
    fence_mbar_init();
  }
  // programmatic dependent of the kernel before it: nothing is read or written before that ends
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- plan: units before each sequence; thread i has sequences [i * per, (i + 1) * per)
  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
  int mine = 0;
  for (int s = s0; s < s1; ++s) mine += seq_of<S>(p, s).units(p.num_kv_heads);
  int before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += v;
  }
  if (lane == 31) sm.scan[warp] = before;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sm.scan[w];
    total += sm.scan[w];
  }
  before -= mine;
  const int ctas = min(static_cast<int>(gridDim.x), total);
  Cut* cuts = reinterpret_cast<Cut*>(p.cuts);
  if (static_cast<int>(blockIdx.x) >= ctas) {
    if (tid == 0) cuts[blockIdx.x].parts = 0;
    return;
  }
  const Ranges ranges(total, ctas);
  const int u0 = ranges.begin(blockIdx.x);
  if (before <= u0 && u0 < before + mine) {
    int at = before;
    int s = s0;
    for (; s < s1; ++s) {
      const int n = seq_of<S>(p, s).units(p.num_kv_heads);
      if (u0 < at + n) break;
      at += n;
    }
    sm.first_seq = s;
    sm.first_unit = at;
  }
  __syncthreads();
  Cursor c;
  c.seq = sm.first_seq;
  c.s = seq_of<S>(p, c.seq);
  {
    const int rest = u0 - sm.first_unit;
    const int each = c.s.tiles + kPieceUnits;
    const int pair = rest / each;
    c.begin = sm.first_unit + pair * each;
    c.rg = pair / p.num_kv_heads;
    c.kvh = pair - c.rg * p.num_kv_heads;
    c.tile = max(0, u0 - c.begin - kPieceUnits);
    c.until = ranges.begin(blockIdx.x + 1);
    c.set_end();
  }
  if (c.tile >= c.end) {  // none but what is counted for a pair beside its tiles
    if (tid == 0) cuts[blockIdx.x].parts = 0;
    return;
  }
  if (warp == kWarps) {
    load<S>(p, map_k, map_v, sm, c, lane);
  } else {
    compute<S>(p, sm, c, ranges, warp, lane);
  }
}

template <typename S>
constexpr int kSmemBytes = static_cast<int>(sizeof(Smem<S>)) + 1024;  // its alignment

template <typename S>
cudaError_t prepare() {
  static_assert(kSmemBytes<S> * S::kCtas <= (227 - (S::kCtas - 1)) * 1024, "shared memory of an SM");
  return cudaFuncSetAttribute(int4_decode_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes<S>);
}

template <typename S>
int resident(int num_sms) {  // CTAs that run at once; asked before the first launch on a device, which it prepares
  int per_sm = 0;
  if (prepare<S>() != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, int4_decode_kernel<S>, kThreads, kSmemBytes<S>) !=
          cudaSuccess)
    return 0;
  return per_sm * num_sms;
}

template <typename S>
cudaError_t launch(Int4AttnParams p, const CUtensorMap& map_k, const CUtensorMap& map_v, int grid, cudaStream_t stream) {
  p.unit_pages = kUnit / p.block_size;
  p.unit_rest = kUnit % p.block_size;
  p.group_inverse = static_cast<uint32_t>(((int64_t{1} << 31) + p.group - 1) / p.group);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes<S>;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, int4_decode_kernel<S>, p, map_k, map_v);
}

// Planes of rows in a row group: as many as the longest chunk's rows need, at most four.
int planes_of(int group, int max_q) {
  const int64_t rows = static_cast<int64_t>(group) * max_q;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : 4;
}

}  // namespace

cudaError_t int4_error_word(void** word) { return cudaGetSymbolAddress(word, g_error); }

int int4_decode_grid(int group, int max_q) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> known[kMaxDevices][5];  // by device and planes; 0: not asked yet
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  const int v = planes_of(group, max_q);
  int n = known[dev][v].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    n = v == 1   ? resident<Shape<1>>(sms)
        : v == 2 ? resident<Shape<2>>(sms)
        : v == 3 ? resident<Shape<3>>(sms)
                 : resident<Shape<4>>(sms);
    known[dev][v].store(n, std::memory_order_relaxed);
  }
  return n;
}

bool int4_decode_fits(int group, int max_q, int num_seqs, int num_kv_heads, int64_t longest) {
  const int rows = 8 * planes_of(group, max_q);
  const int64_t groups = (static_cast<int64_t>(group) * max_q + rows - 1) / rows;
  const int64_t each = (longest / kUnit + 1 + kPieceUnits) * groups * num_kv_heads;  // of a sequence, at most
  return each < INT_MAX && each * num_seqs < INT_MAX;
}

int64_t int4_decode_workspace_bytes(int group, int max_q, int grid) {
  const int64_t part = static_cast<int64_t>(8 * planes_of(group, max_q)) * (kHeadDim + 2) * 4;
  return static_cast<int64_t>(grid) * (kInt4CutBytes + 2 * part);
}

int int4_decode_rows(int group, int max_q) { return 8 * planes_of(group, max_q); }

cudaError_t launch_int4_decode(Int4AttnParams p, const CUtensorMap& map_k, const CUtensorMap& map_v, int grid,
                               cudaStream_t stream) {
  switch (planes_of(p.group, p.max_q)) {
    case 1: return launch<Shape<1>>(p, map_k, map_v, grid, stream);
    case 2: return launch<Shape<2>>(p, map_k, map_v, grid, stream);
    case 3: return launch<Shape<3>>(p, map_k, map_v, grid, stream);
    default: return launch<Shape<4>>(p, map_k, map_v, grid, stream);
  }
}

}  // namespace fp8attn
