// Causal attention of long chunks of new tokens over the paged 4-bit cache, on the tcgen05 tensor cores.
//
// A work item is 256 query rows of one kv head (rows are (token, query head of the group), token by token) in two
// groups of 128, over all positions that they see, 128 at a time.  Both groups use every tile of K and V, and while
// the softmax of one is computed, the tensor cores work for the other:
//   S_g = Q_g K^T        M = N = 128, K = 128: 8 kind::f16 products, Q and K from shared memory
//   P_g = 2^(S_g - m)    f16, over the columns of S_g
//   O_g += P_g V         8 products, P from tensor memory, V from shared memory
// Tiles arrive as codes (17 KB instead of 64) and are turned into f16 once for all 256 rows: a masked pair of codes
// is a pair of f16 numbers (code * 2^-24, or * 2^-20 for the high half of a byte), and one packed multiply-add with
// (step, low) makes the values.  A block of 32 rows of K or V has a power of two that puts its largest value between 2^-7
// and 2^-6, over all of bf16's range; values are rounded once, to 11 bits.  K's power is put back into the block's columns
// of scores.  V's goes into P, whose reference is the query row's own largest p |v| and not its largest p, so that
// what a query row gets does not depend on the size of rows that it does not see.  Within eight values the order is
// 0 4 1 5 2 6 3 7, as the masks give it: q is laid out in the same order, outputs are put back.  A row of K or V that is not
// finite becomes NaN in K and zero in V, so that it reaches just those query rows that see it.
//
// Rows of one block that differ by more than 2^kSpread cannot share a power: the small ones would leave f16's normal numbers
// (below 2^-14).  In such a block each row of K and V has its own, at the cost of a second pass over the tile's scores and a
// second exponential (all tiles of 2,048 of 32,768: 3,540 us for 940; each sequence's first row alone: 950).
//
// Measured for this (2,048 of 32,768 and 7 prompts in us; 915 to 945 and 171 with one power for a tile of K and one that grows for
// V, which small rows do not survive; 937 to 950 and 184 as it is): one power for the four blocks of a tile, agreed on by the
// unpacking warps, 962 and 181; found by each of them, 982 and 185; by a warp of its own, which prepares steps and lowest values
// ahead of them, 1,250 and 234; codes made whole numbers by another f16
// operation, so that a tile has 2^21 more room and rarely needs powers, 1,100 and 193.
//
// Roundings: q is exact; values of K and V 2^-12, P 2^-12, a fourth of the exponentials 1e-4; statistics and sums in fp32, those of
// the tensor cores cut at 2^-24 of their largest term.  Off in the 2-norm: 1.68e-3 (7 prompts) and 1.69e-3 (2,048 of 32,768), of
// which the output's own rounding is 1.66e-3.
//
// Bound by the chain of a group: products of its tile (1,056 cycles: one every 66) behind the other group's, then its
// softmax (about 2,050), 4,100 cycles for a tile of both groups; tensor cores and issue slots are half busy (2,048 new
// tokens of 32,768 positions, 32 heads: 937 to 950 us, 1,130 TFLOP/s).  A softmax row of 128 needs 1,024 cycles of the
// exponential unit for each group, so 1 of 4 pairs takes a polynomial instead (7 prompts: 182 to 176 us).  Tried, when
// these took 910 and 170 us: scores and P by halves of a tile, so that softmax and products of a group overlap (1,404 us: products of 64 columns
// take as long as those of 128), P alone by halves (1,041: the issuing warp waits for one group while the other is
// ready), an issuing warp for each group (1,250), the groups' blocks of products in a loop (941), barriers looked at
// between two blocks (1,107).  Short items (7 prompts) pay 9,000 cycles for q and outputs beside some 4 tiles;
// q brought by bulk copies of 128 bytes took 322 us, by two warps of its own 182, before the outputs of the item before
// it 175; outputs through shared memory 180.
//
// Warps: 0-3 and 4-7 softmax of the groups, a row each thread; 8-11 turn codes into f16; 12 loads (TMA); 13 issues
// the products.  Registers are moved from the others to the softmax (setmaxnreg).  Units of 128 positions of all items
// are cut into equal ranges, one for each SM, and parts of cut items joined by another kernel.
#include "int4_attention.cuh"
#include "tcgen05.cuh"

#include <atomic>
#include <climits>

namespace fp8attn {
namespace {

constexpr int kRows = 128;          // of a group
constexpr int kItem = 2 * kRows;    // rows of a work item
constexpr int kTile = 128;          // positions
constexpr int kPieceUnits = 3;      // what a work item costs beside its tiles, in units of a tile
constexpr int kRaw = 3;             // stages of codes, K 0, K 1, V 0, K 2, V 1, ...
constexpr int kThreads = 512;
constexpr int kUnpackWarp = 8, kLoadWarp = 12, kMmaWarp = 13;
constexpr int kSoftmaxRegs = 184, kUnpackRegs = 88, kOtherRegs = 56;
static_assert(2 * kSoftmaxRegs + kUnpackRegs + kOtherRegs == 4 * 128, "all of the registers, and no more");
constexpr float kSlack = 8.f;  // a reference maximum may lag by 2^8
constexpr float kDown = 1.f / 128.f;  // codes are f16 numbers code * 2^-24: steps of numbers below 2^-6 times 2^24 fit f16
constexpr int kSpread = 6;  // within 2^7 of the largest a row's error is 2^-18 2^6 of its largest value at most: f16's own
constexpr int kBlock = 32;  // rows of K and V that share a power of two
constexpr float kGap = 60.f;  // a block's V may be 2^-60 of a row's reference, so that P of it, of which l is summed, is there
constexpr float kLift = 4.f;   // P and its sums are 2^4 times as large: P between 2^-14 and 2^12 is a normal number
constexpr int kOBytes = kTile * 128;  // a 64-value block of an operand: 128 rows of 128 bytes

struct __align__(1024) Smem {
  uint8_t q[2][2 * kOBytes];   // K-major, 128B swizzle, two blocks of 64 values
  uint8_t k[2][2 * kOBytes];
  uint8_t v[2][2 * kOBytes];   // MN-major, the same layout
  uint8_t raw[kRaw][kTile * 64];  // codes of K or V, 64B swizzle
  uint2 raw_scale[kRaw][kTile];   // beside codes of K: scales of both
  uint32_t raw_there[kRaw];       // and which 16 positions are in pages of the cache
  // of a tile, by unit mod 4, and its blocks: K's power of two (without kDown; negative: each row has its own); the exponent of
  // V's; raw_there; and rows' own powers: their exponents + 127, of K and V
  float4 k_back[4], v_power[4];  // a component for each block
  uint32_t there[4];
  uint16_t powers[4][kTile];
  uint64_t raw_full[kRaw], raw_empty[kRaw];
  uint64_t k_full[2], k_free[2], v_full[2], v_free[2];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t drained;
  int64_t scan[kThreads / 32];
  int first_seq, first_unit;  // the sequence in which the CTA's range begins, its first unit
  uint32_t tmem;
};

struct Seq {
  int q_first, nq, nk, vis, groups;
};

__device__ __forceinline__ Seq seq_of(const Int4AttnParams& p, int s) {
  Seq q;
  q.q_first = __ldg(p.cu_q + s);
  q.nq = __ldg(p.cu_q + s + 1) - q.q_first;
  q.nk = __ldg(p.cu_k + s + 1) - __ldg(p.cu_k + s);
  if (q.nq <= p.min_q || q.nq > p.max_q) q.nq = 0;  // the other kernel's, or nobody's
  q.vis = max(0, min(q.nk, p.max_blocks * p.block_size));
  q.groups = (q.nq * p.group + kItem - 1) / kItem;
  return q;
}
// Row groups of a sequence one after another: how many tiles each sees (those of its last row, and one where it sees
// none: zeros are written), without a division for each.
struct Groups {
  int last, rest;  // token of the group's last row, and what is left of the division
  __device__ __forceinline__ Groups(const Int4AttnParams& p, int rg) {
    const int row = (rg + 1) * kItem - 1;
    last = row / p.group;
    rest = row - last * p.group;
  }
  __device__ __forceinline__ int tiles(const Seq& q) const {
    return max(1, (min(q.vis, min(last, q.nq - 1) + q.nk - q.nq + 1) + kTile - 1) >> 7);
  }
  __device__ __forceinline__ void next(const Int4AttnParams& p) {
    last += p.item_tokens;
    rest += p.item_rest;
    if (rest >= p.group) {
      rest -= p.group;
      ++last;
    }
  }
};
static_assert(kTile == 128 && kTile / kBlock == 4, "the shift in Groups::tiles, Smem's float4");
__device__ __forceinline__ int tiles_of(const Int4AttnParams& p, const Seq& q, int rg) { return Groups(p, rg).tiles(q); }
__device__ __forceinline__ int64_t units_of(const Int4AttnParams& p, const Seq& q) {
  int64_t n = 0;
  Groups at(p, 0);
  for (int rg = 0; rg < q.groups; ++rg) {
    n += at.tiles(q) + kPieceUnits;
    at.next(p);
  }
  return n * p.num_kv_heads;
}

// The piece of a work item that a warp is at: sequence, row group, kv head, its tiles [tile, end) of `tiles`.  An item's
// units are kPieceUnits for what it costs beside its tiles, and then its tiles; a piece is what of it lies in the CTA's
// range, which ends at unit `until`.
struct Cursor {
  int seq, rg, kvh, tile, end, tiles;
  int begin, until;  // the item's first unit
  Seq s;
  // Whether another piece with a tile follows.
  __device__ __forceinline__ bool more() const { return begin + tiles + 2 * kPieceUnits < until; }
  __device__ __forceinline__ void set_end() {
    end = max(0, min(tiles, until - begin - kPieceUnits));
  }
  __device__ __forceinline__ bool whole() const { return tile == 0 && end == tiles; }
};

__device__ __forceinline__ void next_piece(const Int4AttnParams& p, Cursor& c) {
  c.tile = 0;
  c.begin += c.tiles + kPieceUnits;
  if (++c.kvh >= p.num_kv_heads) {
    c.kvh = 0;
    if (++c.rg >= c.s.groups) {
      c.rg = 0;
      do {  // there is one: more()
        c.s = seq_of(p, ++c.seq);
      } while (c.s.groups == 0);
    }
    c.tiles = tiles_of(p, c.s, c.rg);
  }
  c.set_end();
}

__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// kind::f16 with both operands from shared memory.
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// ------------------------------------------------------------------------------------------ loading
// Lane i < 8 looks up the page of positions 16 i of each tile, and the lanes at which a TMA box begins load it.
__device__ __forceinline__ void load_role(const Int4AttnParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v,
                                          Smem& sm, Cursor c, int lane) {
  int column = 0, place = 0;
  auto look_up = [&]() {
    const int pos = c.tile * kTile + lane * 16;
    if (lane >= 8 || pos >= c.s.vis) return -1;
    const int page = ldg_keep(p.block_tables + c.seq * p.bt_stride + column);
    return page >= 0 && page < p.num_blocks ? page : -1;
  };
  auto find = [&]() {
    const int pos = c.tile * kTile + lane * 16;
    column = pos / p.block_size;
    place = pos - column * p.block_size;
    return look_up();
  };
  int page = find();
  int stage = 0, v_row = 0;
  uint32_t round = 0, loaded = 0, v_boxes = 0;
  bool v_mine = false, ok = true;
  const bool begins = lane < 8 && lane % (p.box_rows / 16) == 0;
  // The next stage's barrier, once the stage is free; null when a wait has given up.
  auto take = [&]() -> uint64_t* {
    ok = ok && (round == 0 || wait_all(&sm.raw_empty[stage], (round - 1) & 1u, p.err));
    return ok ? &sm.raw_full[stage] : nullptr;
  };
  auto done = [&]() {
    loaded |= 1u << stage;
    if (++stage == kRaw) {
      stage = 0;
      ++round;
    }
  };
  bool here = true, before = false;  // a unit, and one before it
  while ((here || before) && ok) {
    const int row = (page * p.num_kv_heads + c.kvh) * p.block_size + place;
    const bool mine = begins && page >= 0;
    const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
    const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine)) * p.box_rows;
    const bool k_now = here, v_now = before;
    before = here;
    if (here) {  // the next unit's pages
      if (++c.tile < c.end) {
        column += p.unit_pages;  // whole pages in a tile, and what is left
        place += p.unit_rest;
        if (place >= p.block_size) {
          place -= p.block_size;
          ++column;
        }
        page = look_up();
      } else if (c.more()) {
        next_piece(p, c);
        page = find();
      } else {
        here = false;
      }
    }
    if (k_now) {
      uint64_t* bar = take();
      if (bar == nullptr) break;
      if (lane == 0) {
        sm.raw_there[stage] = there;
        mbar_arrive_expect_tx(bar, boxes * 72);
      }
      __syncwarp();
      if (mine) {
        tma_load_2d(sm.raw[stage] + lane * 1024, &map_k, bar, 0, row);
        bulk_load(smem_u32(sm.raw_scale[stage] + lane * 16), p.kv_scale + static_cast<int64_t>(row) * 4, p.box_rows * 8,
                  bar);
      }
      done();
    }
    if (v_now) {
      uint64_t* bar = take();
      if (bar == nullptr) break;
      if (lane == 0) mbar_arrive_expect_tx(bar, v_boxes * 64);
      __syncwarp();
      if (v_mine) tma_load_2d(sm.raw[stage] + lane * 1024, &map_v, bar, 0, v_row);
      done();
    }
    v_row = row;
    v_mine = mine;
    v_boxes = boxes;
  }
  // copies in flight after a wait that gave up: they must land (or run out of time) before the CTA ends
  if (!ok)
    for (int i = 0; i < kRaw; ++i)
      if (loaded >> i & 1u) wait_all(&sm.raw_full[i], (i < stage ? round : round - 1) & 1u, p.err);
}

// ------------------------------------------------------------------------------------------ codes -> f16
// Eight values (a word of codes) -> four f16 pairs, values 0 4, 1 5, 2 6 and 3 7.
__device__ __forceinline__ uint4 unpack8(uint32_t w, uint32_t even, uint32_t odd, uint32_t low) {
  const uint32_t y = w >> 8;
  return make_uint4(fma_f16x2(w & 0x000F000Fu, even, low), fma_f16x2(w & 0x00F000F0u, odd, low),
                    fma_f16x2(y & 0x000F000Fu, even, low), fma_f16x2(y & 0x00F000F0u, odd, low));
}

__device__ __forceinline__ uint32_t twice_f16(float x) {
  const uint32_t h = __half_as_ushort(__float2half_rn(x));
  return h | h << 16;
}

// What a row's codes are multiplied by (in the low and in the high half of a byte), and its lowest value; f16 twice.
struct RowScale {
  uint32_t even, odd, low;
};
__device__ __forceinline__ RowScale row_scale(float step, float low) {
  return {twice_f16(step * (16777216.f * kDown)), twice_f16(step * (1048576.f * kDown)), twice_f16(low * kDown)};
}
// The power of two that takes a number to between 1 and 2; it and its inverse are normal numbers (the largest and the
// smallest numbers come out up to twice as large, and smaller).
__device__ __forceinline__ int power_of(float x) { return max(-126, min(exponent(x), 126)); }

// K is one tile ahead of V (steps K 0, K 1, V 0, K 2, V 1, ...): the scores of the next tile are never waited for.
// One body for both, so that the loop stays small.
__device__ __forceinline__ void unpack_role(const Int4AttnParams& p, Smem& sm, Cursor c, int warp, int lane) {
  const int g = lane >> 2, t = lane & 3;
  RowScale v_scale = {0, 0, 0}, next_v = {0, 0, 0};
  int stage = 0;
  uint32_t raw_parity = 0;
  int k_unit = 0, v_unit = 0;
  bool more_k = true;
#pragma unroll 1
  for (int step = 0; more_k || v_unit < k_unit; ++step) {
    const bool is_k = more_k && (step == 0 || (step & 1));
    if (!wait_all(&sm.raw_full[stage], raw_parity, p.err)) return;
    RowScale mine = v_scale;
    uint32_t there = 0;
    float k_back = 1.f, v_power = 0.f;
    if (is_k) {
      // ---- the warp's 32 rows, a lane each: the largest and the smallest of those that are there
      there = sm.raw_there[stage];
      const int row = 32 * warp + lane;
      const uint2 sc = sm.raw_scale[stage][row];
      const float ks = __uint_as_float(sc.x << 16), kl = __uint_as_float(sc.x & 0xFFFF0000u);
      const float vs = __uint_as_float(sc.y << 16), vl = __uint_as_float(sc.y & 0xFFFF0000u);
      const float kt = fmaxf(fabsf(kl), fabsf(fmaf(15.f, ks, kl))), vt = fmaxf(fabsf(vl), fabsf(fmaf(15.f, vs, vl)));
      const bool held = (there >> (row >> 4) & 1u) && c.tile * kTile + row < c.s.vis;
      // a sum: NaN and infinity do not get lost; of an eighth each, which numbers cannot bring past fp32's range
      const bool fine = held && fmaf(kt, 0.125f, fmaf(fabsf(ks), 0.125f, fmaf(vt, 0.125f, fabsf(vs) * 0.125f))) < INFINITY;
      const int ke = power_of(kt), ve = power_of(vt);
      const int k_most = __reduce_max_sync(0xffffffffu, fine ? ke : -126), v_most = __reduce_max_sync(0xffffffffu, fine ? ve : -126);
      // small rows.  Zeros are exact with any power, but in V they count: P of the others must not sink beside theirs
      const bool small = fine && ((kt > 0.f && k_most - ke > kSpread) || v_most - ve > kSpread);
      const bool own = __any_sync(0xffffffffu, small);
      const int k_exp = own && fine ? ke : k_most, v_exp = own && fine ? ve : v_most;
      const float k_to = pow2(-k_exp), v_to = pow2(-v_exp);
      mine = fine ? row_scale(ks * k_to, kl * k_to) : row_scale(0.f, held ? __uint_as_float(0x7FC00000u) : 0.f);
      next_v = fine ? row_scale(vs * v_to, vl * v_to) : row_scale(0.f, 0.f);
      if (own) sm.powers[k_unit & 3][row] = static_cast<uint16_t>((k_exp + 127) | (v_exp + 127) << 8);
      k_back = own ? -1.f : pow2(k_most);
      // a block without rows: the largest power, so that it is never a row's smallest
      v_power = __any_sync(0xffffffffu, fine) ? static_cast<float>(v_most) : 126.f;
    }
    // ---- 32 rows of codes (lane: rows 8 i + g, 16-byte piece t) into the operand
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 32 * warp + 8 * i + g;
      x[i] = ld_shared_v4(smem_u32(sm.raw[stage]) + row * 64 + ((t ^ (row >> 1 & 3)) * 16));
    }
    const int unit = is_k ? k_unit : v_unit;
    const int buf = unit & 1;
    // its last readers
    if (unit > 1 && !wait_all(is_k ? &sm.k_free[buf] : &sm.v_free[buf], static_cast<uint32_t>((unit >> 1) - 1) & 1u, p.err))
      return;
    const uint32_t dst = smem_u32(is_k ? sm.k[buf] : sm.v[buf]) + (t >> 1) * kOBytes;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 32 * warp + 8 * i + g;
      const uint32_t a = __shfl_sync(0xffffffffu, mine.even, 8 * i + g), b = __shfl_sync(0xffffffffu, mine.odd, 8 * i + g);
      const uint32_t d = __shfl_sync(0xffffffffu, mine.low, 8 * i + g);
      // pieces 2 and 3 (the second block of values) in another order: no bank conflicts
      const bool swap = t & 2;
      const uint32_t w[4] = {swap ? x[i].z : x[i].x, swap ? x[i].w : x[i].y, swap ? x[i].x : x[i].z, swap ? x[i].y : x[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 y = unpack8(w[k], a, b, d);
        const int chunk = (t & 1) * 4 + (k ^ (t & 2));
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + row * 128 + ((chunk ^ (row & 7)) * 16)), "r"(y.x),
                     "r"(y.y), "r"(y.z), "r"(y.w));
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (is_k) {
        const int slot = k_unit & 3;
        reinterpret_cast<float*>(&sm.k_back[slot])[warp] = k_back;
        reinterpret_cast<float*>(&sm.v_power[slot])[warp] = v_power;
        if (warp == 0) sm.there[slot] = there;
      }
      mbar_arrive(is_k ? &sm.k_full[buf] : &sm.v_full[buf]);
      mbar_arrive(&sm.raw_empty[stage]);
    }
    if (++stage == kRaw) {
      stage = 0;
      raw_parity ^= 1u;
    }
    if (is_k) {
      ++k_unit;
      if (++c.tile == c.end) {
        more_k = c.more();
        if (more_k) next_piece(p, c);
      }
    } else {
      ++v_unit;
    }
    if (!is_k || step == 0) v_scale = next_v;
  }
}

// ------------------------------------------------------------------------------------------ products
// The whole warp goes through the loop, so that descriptors and addresses are uniform, and one lane issues.
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
  return chosen != 0;
}

__device__ __forceinline__ void mma_role(const Int4AttnParams& p, Smem& sm, Cursor c) {
  constexpr uint32_t idesc_s = tc::idesc_f16(128, 128, false, false), idesc_pv = tc::idesc_f16(128, 128, false, true);
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  const uint64_t dq = tc::smem_desc(smem_u32(sm.q[0]), 16, 1024, tc::kSw128);
  const uint64_t dk = tc::smem_desc(smem_u32(sm.k[0]), 16, 1024, tc::kSw128);
  const uint64_t dv = tc::smem_desc(smem_u32(sm.v[0]), kOBytes, 1024, tc::kSw128);
  uint32_t q_parity = 0, p_parity = 0;
  bool ok = true;
  for (int u = 0; ok;) {
    const int n = c.end - c.tile;
    const int groups = c.s.nq * p.group - c.rg * kItem > kRows ? 2 : 1;
#pragma unroll 1
    for (int i = 0; i <= n && ok; ++i) {
      const int at = u + i;  // scores of this unit, values of the one before it
      const int k_buf = at & 1, v_buf = (at - 1) & 1;
      const uint64_t v_desc = dv + static_cast<uint64_t>(v_buf * (2 * kOBytes >> 4));
      const uint64_t k_desc = dk + static_cast<uint64_t>(k_buf * (2 * kOBytes >> 4));
      uint64_t* const v_free = &sm.v_free[v_buf];
      uint64_t* const k_free = &sm.k_free[k_buf];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (g >= groups) break;
        // all that the group's products wait for, and then all of them: the tensor cores run dry between two blocks
        if (g == 0) {
          if (i > 0) ok = wait_all(&sm.v_full[v_buf], static_cast<uint32_t>((at - 1) >> 1) & 1u, p.err);
          if (i < n) ok = ok && wait_all(&sm.k_full[k_buf], static_cast<uint32_t>(at >> 1) & 1u, p.err);
        }
        if (i == 0) ok = ok && wait_all(&sm.q_full[g], q_parity >> g & 1u, p.err);
        if (i > 0) {
          ok = ok && wait_all(&sm.p_full[g], p_parity >> g & 1u, p.err);
          p_parity ^= 1u << g;
        }
        if (!ok) break;
        tc::fence_after_sync();
        if (elect_one()) {
          if (i > 0) {  // O_g += P_g V, 16 positions at a time: V's rows are 128 bytes
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
              tc::mma_f16_ts(tmem + 256 * g + 128, tmem + 256 * g + 8 * k,
                             v_desc + static_cast<uint64_t>(k * (16 * 128 >> 4)), idesc_pv, i > 1 || k > 0 ? 1u : 0u);
            if (i == n) tc::commit(&sm.o_full[g]);
            if (g == groups - 1) tc::commit(v_free);
          }
          if (i < n) {
            const uint64_t a = dq + static_cast<uint64_t>(g * (2 * kOBytes >> 4));
#pragma unroll
            for (int k = 0; k < 8; ++k) {  // 16 values: 32 bytes, four to a block
              const uint64_t step = static_cast<uint64_t>((k >> 2) * (kOBytes >> 4) + (k & 3) * 2);
              mma_f16_ss(tmem + 256 * g, a + step, k_desc + step, idesc_s, k > 0 ? 1u : 0u);
            }
            tc::commit(&sm.s_full[g]);
            if (g == groups - 1) tc::commit(k_free);
          }
        }
        __syncwarp();
      }
    }
    q_parity ^= groups == 2 ? 3u : 1u;
    u += n;
    if (!c.more()) break;
    next_piece(p, c);
  }
  if (!ok) {  // products in flight must end before the CTA does
    if (elect_one()) tc::commit(&sm.drained);
    wait_all(&sm.drained, 0, p.err);
  }
}

// ------------------------------------------------------------------------------------------ softmax
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// 32 bytes; wide: on a boundary of 32 (else of 16).
__device__ __forceinline__ void st_global_32(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f,
                                             uint32_t g, uint32_t h, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e),
                 "r"(f), "r"(g), "r"(h)
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(a, b, c, d);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(e, f, g, h);
  }
}

// Rows of a work item, every other one: row of the kv head, its token's row of q and its query head.
struct Walk {
  int row, head, in_group;
  int64_t token;
  __device__ __forceinline__ Walk(const Int4AttnParams& p, const Cursor& c, int in_item) {
    row = c.rg * kItem + in_item;
    const int t = row / p.group;
    in_group = row - t * p.group;
    head = c.kvh * p.group + in_group;
    token = static_cast<int64_t>(c.s.q_first) + t;
  }
  __device__ __forceinline__ void two_on(const Int4AttnParams& p) {
    row += 2;
    token += p.two_tokens;
    in_group += p.two_heads;
    head += p.two_heads;
    if (in_group >= p.group) {
      in_group -= p.group;
      head -= p.group;
      ++token;
    }
  }
};

// Which of the columns c0 .. c0 + 31 of a tile a row sees: in pages that are there, and below `seen`.
__device__ __forceinline__ uint32_t seen_of(uint32_t there, int seen, int c0) {
  const uint32_t part = there >> (c0 >> 4);
  const uint32_t held = ((part & 1u) ? 0xFFFFu : 0u) | ((part & 2u) ? 0xFFFF0000u : 0u);
  const int left = seen - c0;
  return held & (left >= 32 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << left) - 1u);
}

// Minus infinity for the columns that a row does not see.
__device__ __forceinline__ void hide(uint32_t (&w)[4][32], uint32_t there, int seen) {
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const uint32_t mask = seen_of(there, seen, 32 * h);
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (!(mask >> k & 1u)) w[h][k] = 0xFF800000u;
  }
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The 16-byte piece of a 256-byte row in a group's q.
__device__ __forceinline__ uint32_t q_piece(uint32_t q, int row, int piece) {
  return q + (piece >> 3) * kOBytes + row * 128 + (((piece & 7) ^ (row & 7)) * 16);
}

// A row's references: m of its largest score, and power, 2^power being its largest p |v| so far.
struct Reference {
  float m, power;
  // New ones where they lag too far (also for NaN: the row's sums and outputs become NaN).
  __device__ __forceinline__ Reference after(float top, float top_v) const {
    const bool higher = !(top <= m + kSlack);
    const float now = higher ? top : m;
    return {now, higher || top_v - now > power + kSlack ? ceilf(fmaxf(power + (m - now), top_v - now)) : power};
  }
};

// O's row in tensor memory, times f.
__device__ __forceinline__ void scale_o(uint32_t o_tmem, float f) {
#pragma unroll 1
  for (int c0 = 0; c0 < kHeadDim; c0 += 8) {
    float y[8];
    tc::ld8(o_tmem + c0, y);
    tc::wait_ld();
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] *= f;
    tc::st8(o_tmem + c0, y);
  }
}

// A tile with rows that have powers of their own, or blocks of V that differ by more than 2^kGap:
// l's terms 2^(score - m + kLift) and P = 2^(score - m + kLift - power) of V's power are exponentials for themselves.
__device__ __noinline__ float3 wide_tile(const Smem& sm, uint32_t s_tmem, float cs, int slot, uint32_t there, int seen, bool rest,
                                       Reference at, float l) {
  // 32 scores, -infinity where the row does not see one; v: exponents of V's powers
  auto scores = [&](int h, float (&x)[32], float (&v)[32]) {
    uint32_t w[32];
    tmem_ld32(s_tmem + 32 * h, w);
    tc::wait_ld();
    const uint32_t mask = seen_of(there, seen, 32 * h);
    const float back = reinterpret_cast<const float*>(&sm.k_back[slot])[h];
    const float v_power = reinterpret_cast<const float*>(&sm.v_power[slot])[h];
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const int own = sm.powers[slot][32 * h + k];
      const float k_back = back < 0.f ? pow2((own & 255) - 127) : back;
      v[k] = back < 0.f ? static_cast<float>((own >> 8) - 127) : v_power;
      x[k] = mask >> k & 1u ? __uint_as_float(w[k]) * (cs * k_back) : -INFINITY;
    }
  };
  float top = -INFINITY, top_v = -INFINITY;
#pragma unroll 1
  for (int h = 0; h < 4; ++h) {
    float x[32], v[32];
    scores(h, x, v);
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      top = max3_nan(top, x[k], x[k]);
      top_v = fmaxf(top_v, x[k] + v[k]);
    }
  }
  const Reference to = at.after(top, top_v);
  const float f = ex2((at.m - to.m) + (at.power - to.power));
  l *= ex2(at.m - to.m);
  at = to;
  if (rest && __any_sync(0xffffffffu, f != 1.f)) scale_o(s_tmem + 128, f);
  float sum = 0.f;
#pragma unroll 1
  for (int h = 0; h < 4; ++h) {  // P's columns lie over those of S that have been read
    float x[32], v[32];
    scores(h, x, v);
    uint32_t pw[16];
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
      const float a = x[k] - at.m + kLift, b = x[k + 1] - at.m + kLift;
      sum += ex2(a) + ex2(b);
      pw[k / 2] = pack_f16x2(ex2(a + (v[k] - at.power)), ex2(b + (v[k + 1] - at.power)));
    }
    tc::st16u(s_tmem + 16 * h, pw);
  }
  return make_float3(at.m, at.power, l + sum);
}

__device__ __forceinline__ void softmax_role(const Int4AttnParams& p, Smem& sm, Cursor next, const Ranges& ranges,
                                             int g, int tid) {
  const int r = tid & 127, warp = r >> 5, lane = tid & 31;
  const uint32_t s_tmem = sm.tmem + (static_cast<uint32_t>(32 * warp) << 16) + 256 * g, o_tmem = s_tmem + 128;
  const uint32_t q = smem_u32(sm.q[g]);
  uint32_t s_parity = 0, o_parity = 0;
  constexpr int kPart = kItem * (kHeadDim + 2);
  bool first_piece = true;
  Cursor c = next;
  bool started = false, more = true;
  for (int u = 0, n = 0;;) {
    const int rows = c.s.nq * p.group;
    const bool active = started && rows - c.rg * kItem > g * kRows;
    Reference at = {kNone, 0.f};
    float l = 0.f;  // sum of 2^(score - m + kLift); O: of 2^(score - m - power + kLift) v kDown
    if (active) {
      const int row = c.rg * kItem + g * kRows + r;
      const int token = row / p.group;
      const int limit = row < rows ? min(c.s.vis, token + c.s.nk - c.s.nq + 1) : c.s.vis;  // no row: zeros that see anything
      // ---- q: each thread turns its row into f16; a power of two puts the largest value between 2^13 and 2^14
      // A warp brings its 32 rows two at a time, 16 lanes to a row: whole lines.
      {
        Walk at(p, c, g * kRows + 32 * warp + (lane >> 4));
#pragma unroll 2
        for (int i = 0; i < 16; ++i) {
          cp_async16(q_piece(q, 32 * warp + 2 * i + (lane >> 4), lane & 15),
                     p.q + at.token * p.q_row_stride + at.head * kHeadDim + 8 * (lane & 15), at.row < rows);
          at.two_on(p);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
      }
      uint32_t top_bits = 0;  // bf16 magnitudes in order as integers, two at a time
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const uint4 w = ld_shared_v4(q_piece(q, r, i));
        top_bits = __vmaxu2(__vmaxu2(top_bits, w.x & 0x7FFF7FFFu), w.y & 0x7FFF7FFFu);
        top_bits = __vmaxu2(__vmaxu2(top_bits, w.z & 0x7FFF7FFFu), w.w & 0x7FFF7FFFu);
      }
      const float amax = __uint_as_float(max(top_bits & 0xFFFFu, top_bits >> 16) << 16);
      const int e = amax > 0.f && amax < INFINITY ? max(-113, exponent(amax)) - 13 : 0;
      const float to = p.scale_log2 < 0.f ? -pow2(-e) : pow2(-e);  // a negative scale turns q around
      const float cs = fabsf(p.scale_log2) * pow2(e + 7);  // with K's kDown
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const uint4 raw_w = ld_shared_v4(q_piece(q, r, i));
        const uint32_t w[4] = {raw_w.x, raw_w.y, raw_w.z, raw_w.w};
        float x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[2 * k] = __uint_as_float(w[k] << 16) * to;
          x[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u) * to;
        }
        // values 8 i .. 8 i + 7 in the order 0 4 1 5 2 6 3 7
        st_shared_v4(q_piece(q, r, i), pack_f16x2(x[0], x[4]), pack_f16x2(x[1], x[5]), pack_f16x2(x[2], x[6]),
                     pack_f16x2(x[3], x[7]));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[g]);

      for (int i = 0; i < n; ++i) {
        const int slot = (u + i) & 3;
        // S_g of this tile done: so is O_g of the one before it
        if (!wait_all(&sm.s_full[g], s_parity, p.err)) return;
        s_parity ^= 1u;
        tc::fence_after_sync();
        const uint32_t there = sm.there[slot];
        const int seen = limit - (c.tile + i) * kTile;  // columns below this one
        const float4 k_back = sm.k_back[slot], v_power = sm.v_power[slot];
        // up to this score the references stay; NaN: not a tile for what follows
        const float v_least = fminf(fminf(v_power.x, v_power.y), fminf(v_power.z, v_power.w));
        const float v_most = fmaxf(fmaxf(v_power.x, v_power.y), fmaxf(v_power.z, v_power.w));
        const bool own = fminf(fminf(k_back.x, k_back.y), fminf(k_back.z, k_back.w)) < 0.f;
        const float stay = own || at.power - v_least > kGap ? NAN : at.m + fminf(kSlack, at.power + kSlack - v_most);
        // never 0, so that what is not seen (minus infinity) stays so; products are below 2^16
        const float ct[4] = {fmaxf(cs * k_back.x, 1.0e-30f), fmaxf(cs * k_back.y, 1.0e-30f),
                             fmaxf(cs * k_back.z, 1.0e-30f), fmaxf(cs * k_back.w, 1.0e-30f)};
        const bool masked = !__all_sync(0xffffffffu, there == 0xFFu && seen >= kTile);
        uint32_t w[4][32];
#pragma unroll
        for (int h = 0; h < 4; ++h) tmem_ld32(s_tmem + 32 * h, w[h]);
        tc::wait_ld();
        if (masked) hide(w, there, seen);
        // ---- the blocks' maxima; NaN where the row sees one
        float t[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          t[h] = -INFINITY;
#pragma unroll
          for (int k = 0; k < 32; k += 2) t[h] = max3_nan(t[h], __uint_as_float(w[h][k]), __uint_as_float(w[h][k + 1]));
          t[h] *= ct[h];
        }
        const float top = max3_nan(max3_nan(t[0], t[1], t[2]), t[3], t[3]);
        bool wide = false;
        if (!__all_sync(0xffffffffu, top <= stay)) {
          const Reference to = at.after(
              top, fmaxf(fmaxf(t[0] + v_power.x, t[1] + v_power.y), fmaxf(t[2] + v_power.z, t[3] + v_power.w)));
          wide = __any_sync(0xffffffffu, own || to.power - v_least > kGap);
          if (!wide) {
            const float f = ex2((at.m - to.m) + (at.power - to.power));
            l *= ex2(at.m - to.m);
            at = to;
            if (i > 0 && __any_sync(0xffffffffu, f != 1.f)) scale_o(o_tmem, f);
          }
        }
        if (wide) {
          const float3 y = wide_tile(sm, s_tmem, cs, slot, there, seen, i > 0, at, l);
          at = {y.x, y.y};
          l = y.z;
        } else {
          // ---- P over the columns of S, all of which have been read
          const float ev[4] = {v_power.x - at.power, v_power.y - at.power, v_power.z - at.power, v_power.w - at.power};
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const float bias = kLift - at.m + ev[h];
            const uint64_t ct2 = f2_pack(ct[h], ct[h]), bias2 = f2_pack(bias, bias);
            uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
            uint32_t pw[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float x0, x1, p0, p1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(w[h][2 * k]), __uint_as_float(w[h][2 * k + 1])), ct2, bias2), x0, x1);
              if (k % 4 == 3) {
                exp2_poly_x2(x0, x1, p0, p1);
              } else {
                p0 = ex2(x0);
                p1 = ex2(x1);
              }
              sum[k & 1] = f2_add(sum[k & 1], f2_pack(p0, p1));
              pw[k] = pack_f16x2(p0, p1);
            }
            tc::st16u(s_tmem + 16 * h, pw);
            float a0, a1;
            f2_unpack(f2_add(sum[0], sum[1]), a0, a1);
            l = fmaf(a0 + a1, ex2(-ev[h]), l);
          }
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if ((tid & 31) == 0) mbar_arrive(&sm.p_full[g]);
      }
    }
    // ---- the next piece's q on its way to L2
    if (more) {
      const int next_row = min(next.rg * kItem + g * kRows + r, next.s.nq * p.group - 1), next_token = next_row / p.group;
      const uint16_t* src = p.q + (static_cast<int64_t>(next.s.q_first) + next_token) * p.q_row_stride +
                            (next.kvh * p.group + next_row - next_token * p.group) * kHeadDim;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
      asm volatile("prefetch.global.L2 [%0];" ::"l"(src + 64));
    }
    // ---- the piece's end
    if (active) {
      if (!wait_all(&sm.o_full[g], o_parity, p.err)) return;
      o_parity ^= 1u;
      tc::fence_after_sync();
      const bool whole = c.whole();
      // V's power / kDown / l might pass fp32's range where the outputs do not
      const float over = at.power > 100.f ? 16.f : at.power < -100.f ? -16.f : 0.f;
      if (__any_sync(0xffffffffu, over != 0.f)) {
        scale_o(o_tmem, pow2(static_cast<int>(over)));
        tc::wait_st();
      }
      const float back = pow2(max(-126, min(static_cast<int>(at.power - over), 126)));
      const float f = at.m == kNone ? 0.f : __fdiv_rn(back * (1.f / kDown), l);  // 0 for a row that sees nothing
      // a thread stores its row, 32 bytes at a time: whole sectors
      const int row = c.rg * kItem + g * kRows + r, token = row / p.group;
      float* part = p.partials + (2 * static_cast<int64_t>(blockIdx.x) + (first_piece ? 0 : 1)) * kPart;
      uint16_t* const out = p.out + (static_cast<int64_t>(c.s.q_first) + token) * p.out_row_stride +
                            (c.kvh * p.group + row - token * p.group) * kHeadDim;
      uint8_t* dst = whole ? reinterpret_cast<uint8_t*>(out)
                           : reinterpret_cast<uint8_t*>(part + (g * kRows + r) * kHeadDim);
      const bool wide = __all_sync(0xffffffffu, (reinterpret_cast<uintptr_t>(dst) & 31) == 0);
#pragma unroll 1
      for (int c0 = 0; c0 < kHeadDim; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(o_tmem + c0, v);
        tc::wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
        if (whole) {  // back from the order 0 4 1 5 2 6 3 7
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              w[k / 2 + 2 * x] = pack_bf16x2(__uint_as_float(v[k + x]), __uint_as_float(v[k + x + 2]));
              w[k / 2 + 2 * x + 1] = pack_bf16x2(__uint_as_float(v[k + x + 4]), __uint_as_float(v[k + x + 6]));
            }
          }
          if (row < rows) {
            st_global_32(dst + 2 * c0, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], wide);
            st_global_32(dst + 2 * c0 + 32, w[8], w[9], w[10], w[11], w[12], w[13], w[14], w[15], wide);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            st_global_32(dst + 4 * (c0 + k), v[k], v[k + 2], v[k + 4], v[k + 6], v[k + 1], v[k + 3], v[k + 5], v[k + 7],
                         wide);
        }
      }
      if (!whole)
        *reinterpret_cast<float2*>(part + kItem * kHeadDim + 2 * (g * kRows + r)) = make_float2(at.m, at.m == kNone ? 0.f : l);
      tc::fence_before_sync();  // O has been read before the next piece's first P is announced
    }
    if (!more) {
      if (tid == 0) {
        Cut cut = {};
        if (c.tile == 0 && c.end < c.tiles) {
          const int first = c.begin + kPieceUnits, last = first + c.tiles - 1;  // its tiles, as units
          cut.parts = ranges.owner(last) - ranges.owner(first) + 1;
          cut.slot = 2 * blockIdx.x + (first_piece ? 0 : 1);
          cut.rows = min(kItem, rows - c.rg * kItem);
          cut.first_row = c.rg * kItem;
          cut.token = c.s.q_first;
          cut.head = c.kvh * p.group;
        }
        reinterpret_cast<Cut*>(p.cuts)[blockIdx.x] = cut;
      }
      return;
    }
    u += n;
    first_piece = !started;
    started = true;
    c = next;
    n = c.end - c.tile;
    more = c.more();
    if (more) next_piece(p, next);
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    int4_prefill_kernel(const __grid_constant__ Int4AttnParams p, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v) {
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + (1024 - smem_u32(smem_raw) % 1024) % 1024);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kRaw; ++i) {
      mbar_init(&sm.raw_full[i], 1);
      mbar_init(&sm.raw_empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.k_full[i], 4);
      mbar_init(&sm.k_free[i], 1);
      mbar_init(&sm.v_full[i], 4);
      mbar_init(&sm.v_free[i], 1);
      mbar_init(&sm.q_full[i], 4);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.o_full[i], 1);
    }
    mbar_init(&sm.drained, 1);
    fence_mbar_init();
  }
  // programmatic dependent of the kernel before it: nothing is read or written before that ends
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- plan: units before each sequence; thread i has sequences [i * per, (i + 1) * per)
  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += units_of(p, seq_of(p, s));
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
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sm.scan[w];
    total += sm.scan[w];
  }
  before -= mine;
  // Nothing to be joined until the CTA's last piece says so: the joining kernel reads this of every CTA, of one as well
  // whose waits have given up, and the workspace holds anything.
  if (tid == 0) reinterpret_cast<Cut*>(p.cuts)[blockIdx.x].parts = 0;
  if (total > INT_MAX) {  // hours of work: what follows counts in 32 bits
    if (tid == 0) atomicExch(p.err, kDevErrTooLarge);
    return;
  }
  const int ctas = min(static_cast<int>(gridDim.x), static_cast<int>(total));
  if (static_cast<int>(blockIdx.x) >= ctas) return;
  const Ranges ranges(static_cast<int>(total), ctas);
  const int u0 = ranges.begin(blockIdx.x), u1 = ranges.begin(blockIdx.x + 1);
  if (before <= u0 && u0 < before + mine) {
    int64_t at = before;
    int s = s0;
    for (; s < s1; ++s) {
      const int64_t n = units_of(p, seq_of(p, s));
      if (u0 < at + n) break;
      at += n;
    }
    sm.first_seq = s;
    sm.first_unit = static_cast<int>(at);
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(&sm.tmem, 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  Cursor c;
  c.seq = sm.first_seq;
  c.s = seq_of(p, c.seq);
  {
    c.begin = sm.first_unit;
    Groups at(p, 0);
    for (c.rg = 0;; ++c.rg) {
      c.tiles = at.tiles(c.s);
      const int of_group = (c.tiles + kPieceUnits) * p.num_kv_heads;
      if (u0 < c.begin + of_group) break;
      c.begin += of_group;
      at.next(p);
    }
    c.kvh = (u0 - c.begin) / (c.tiles + kPieceUnits);
    c.begin += c.kvh * (c.tiles + kPieceUnits);
    c.tile = max(0, u0 - c.begin - kPieceUnits);
    c.until = u1;
    c.set_end();
  }
  if (c.tile >= c.end) {
    // none but what is counted for an item beside its tiles
  } else if (warp < kUnpackWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    softmax_role(p, sm, c, ranges, warp >> 2, tid);
  } else if (warp < kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUnpackRegs));
    unpack_role(p, sm, c, warp - kUnpackWarp, lane);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kLoadWarp) {
      load_role(p, map_k, map_v, sm, c, lane);
    } else if (warp == kMmaWarp) {
      mma_role(p, sm, c);
    }
    __syncwarp();
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tc::tmem_dealloc(sm.tmem, 512);
}

constexpr int kSmemBytes = static_cast<int>(sizeof(Smem)) + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory of an SM");

}  // namespace

static_assert(kItem == kInt4LongRows, "the joining kernel's rows");

int64_t int4_prefill_workspace_bytes(int num_sms) {
  return static_cast<int64_t>(num_sms) * (kInt4CutBytes + 2ll * kItem * (kHeadDim + 2) * 4);
}

cudaError_t launch_int4_prefill(Int4AttnParams p, const CUtensorMap& map_k, const CUtensorMap& map_v, int num_sms,
                                cudaStream_t stream) {
  p.item_tokens = kItem / p.group;
  p.item_rest = kItem % p.group;
  p.two_tokens = 2 / p.group;
  p.two_heads = 2 % p.group;
  p.unit_pages = kTile / p.block_size;
  p.unit_rest = kTile % p.block_size;
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> prepared[kMaxDevices];  // the kernel's shared memory asked for, once on each device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kMaxDevices || !prepared[dev].load(std::memory_order_relaxed)) {
    e = cudaFuncSetAttribute(int4_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) prepared[dev].store(true, std::memory_order_relaxed);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(num_sms));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, int4_prefill_kernel, p, map_k, map_v);
}

}  // namespace fp8attn
