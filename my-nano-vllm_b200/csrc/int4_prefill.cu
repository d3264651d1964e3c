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
// (step, low) makes the values.  A power of two for each tile of K (taken back in the scores) and one that only
// grows for V (taken back at the end) put the largest value of a tile between 2^-7 and 2^-6, so that any bf16 cache
// fits f16; values are rounded once, to 11 bits.  Within eight values the order is 0 4 1 5 2 6 3 7, as the masks give
// it: q is laid out in the same order, outputs are put back.  A row of K or V that is not finite becomes NaN in K
// and zero in V, so that it reaches just those query rows that see it.
//
// Tensor work: 2 * 2 * 128 * 128 * 256 flop in 2,048 cycles a tile (4,096 multiply-adds a cycle and SM); a softmax
// row of 128 needs 1,024 cycles of the exponential unit for each group, so 5 of 16 pairs take a polynomial instead.
//
// Warps: 0-3 and 4-7 softmax of the groups, a row each thread; 8-11 turn codes into f16; 12 loads (TMA); 13 issues
// the products.  Registers are moved from the others to the softmax (setmaxnreg).  Units of 128 positions of all items
// are cut into equal ranges, one for each SM, and parts of cut items joined by another kernel.
#include "int4_attention.cuh"
#include "tcgen05.cuh"

#include <climits>

namespace fp8attn {
namespace {

constexpr int kRows = 128;          // of a group
constexpr int kItem = 2 * kRows;    // rows of a work item
constexpr int kTile = 128;          // positions
constexpr int kRaw = 3;             // stages of codes
constexpr int kThreads = 512;
constexpr int kUnpackWarp = 8, kLoadWarp = 12, kMmaWarp = 13;
constexpr int kSoftmaxRegs = 184, kUnpackRegs = 88, kOtherRegs = 56;
static_assert(2 * kSoftmaxRegs + kUnpackRegs + kOtherRegs == 4 * 128, "all of the registers, and no more");
constexpr float kSlack = 8.f;  // a reference maximum may lag by 2^8
constexpr float kLift = 4.f;   // P and its sums are 2^4 times as large: P between 2^-14 and 2^12 is a normal number
constexpr int kOBytes = kTile * 128;  // a 64-value block of an operand: 128 rows of 128 bytes

constexpr uint32_t kWild = 1u << 8;   // beside the eight parts of a tile: it has rows that are not finite

struct __align__(1024) Smem {
  uint8_t q[2][2 * kOBytes];   // K-major, 128B swizzle, two blocks of 64 values
  uint8_t k[2][2 * kOBytes];
  uint8_t v[2 * kOBytes];      // MN-major, the same layout
  uint8_t raw_k[kRaw][kTile * 64];  // codes, 64B swizzle
  uint8_t raw_v[kRaw][kTile * 64];
  uint2 raw_scale[kRaw][kTile];
  uint32_t raw_there[kRaw];    // which 16 positions are in pages of the cache
  // of a tile, by unit mod 4: its power of two of K; what V's power changes O by; V's power; raw_there
  float k_back[4], v_change[4], v_back[4];
  uint32_t there[4];
  uint64_t raw_full[kRaw], raw_empty[kRaw];
  uint64_t k_full[2], k_free[2], v_full, v_free;
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t drained;
  int64_t scan[kThreads / 32];
  int64_t first_unit;  // of the sequence in which the CTA's range begins
  int first_seq;
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
// Tiles that a row group sees: those of its last row, and one where it sees none (zeros are written).
__device__ __forceinline__ int tiles_of(const Int4AttnParams& p, const Seq& q, int rg) {
  const int last = (min(q.nq * p.group, (rg + 1) * kItem) - 1) / p.group;
  return max(1, (min(q.vis, last + q.nk - q.nq + 1) + kTile - 1) / kTile);
}
__device__ __forceinline__ int64_t units_of(const Int4AttnParams& p, const Seq& q) {
  int64_t n = 0;
  for (int rg = 0; rg < q.groups; ++rg) n += tiles_of(p, q, rg);
  return n * p.num_kv_heads;
}

// Where in the order of units a warp is: sequence, row group, kv head, tile.
struct Cursor {
  int seq, rg, kvh, tile, tiles;
  Seq s;
};

__device__ __forceinline__ void next_pair(const Int4AttnParams& p, Cursor& c) {
  c.tile = 0;
  if (++c.kvh < p.num_kv_heads) return;
  c.kvh = 0;
  if (++c.rg >= c.s.groups) {
    c.rg = 0;
    do {
      if (++c.seq >= p.num_seqs) return;
      c.s = seq_of(p, c.seq);
    } while (c.s.groups == 0);
  }
  c.tiles = tiles_of(p, c.s, c.rg);
}

__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, int* err) {
  return mbar_wait(bar, parity, err);
}

__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
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
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// ------------------------------------------------------------------------------------------ loading
// Lane i < 8 looks up the page of positions 16 i of each tile, and the lanes at which a TMA box begins load it.
__device__ __forceinline__ void load_role(const Int4AttnParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v,
                                          Smem& sm, Cursor c, int64_t units, int lane) {
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
  int stage = 0;
  uint32_t round = 0, loaded = 0;
  const bool begins = lane < 8 && lane % (p.box_rows / 16) == 0;
  bool ok = true;
  for (int64_t u = 0; u < units; ++u) {
    const int row = (page * p.num_kv_heads + c.kvh) * p.block_size + place;
    const bool mine = begins && page >= 0;
    const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
    const int boxes = __popc(__ballot_sync(0xffffffffu, mine));
    if (u + 1 < units) {  // the next unit's pages
      if (++c.tile < c.tiles) {
        column += p.unit_pages;  // whole pages in a tile, and what is left
        place += p.unit_rest;
        if (place >= p.block_size) {
          place -= p.block_size;
          ++column;
        }
        page = look_up();
      } else {
        next_pair(p, c);
        page = find();
      }
    }
    if (round > 0) ok = wait_all(&sm.raw_empty[stage], (round - 1) & 1u, p.err);
    if (!ok) break;
    uint64_t* bar = &sm.raw_full[stage];
    if (lane == 0) {
      sm.raw_there[stage] = there;
      mbar_arrive_expect_tx(bar, boxes * p.box_rows * 136);
    }
    __syncwarp();
    if (mine) {
      tma_load_2d(sm.raw_k[stage] + lane * 1024, &map_k, bar, 0, row);
      tma_load_2d(sm.raw_v[stage] + lane * 1024, &map_v, bar, 0, row);
      bulk_load(smem_u32(sm.raw_scale[stage] + lane * 16), p.kv_scale + static_cast<int64_t>(row) * 4, p.box_rows * 8,
                bar);
    }
    loaded |= 1u << stage;
    if (++stage == kRaw) {
      stage = 0;
      ++round;
    }
  }
  // copies in flight after a wait that gave up: they must land (or run out of time) before the CTA ends
  if (!ok)
    for (int i = 0; i < kRaw; ++i)
      if (loaded >> i & 1u) wait_all(&sm.raw_full[i], (i < stage ? round : round - 1) & 1u, p.err);
}

// ------------------------------------------------------------------------------------------ codes -> f16
// Eight rows of codes (lane: row g, 16-byte piece t) -> f16 rows of an operand, value = low + step code times 2^-e.
__device__ __forceinline__ void unpack_rows(uint32_t raw, uint32_t dst, int row, int t, uint32_t even, uint32_t odd,
                                            uint32_t low) {
  const uint4 x = ld_shared_v4(raw + row * 64 + ((t ^ (row >> 1 & 3)) * 16));
  // pieces 2 and 3 (the second block of values) in another order: no bank conflicts
  const bool swap = t & 2;
  const uint32_t w[4] = {swap ? x.z : x.x, swap ? x.w : x.y, swap ? x.x : x.z, swap ? x.y : x.w};
  const uint32_t out = dst + (t >> 1) * kOBytes + row * 128;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t y = w[i] >> 8;
    const uint32_t a = fma_f16x2(w[i] & 0x000F000Fu, even, low), b = fma_f16x2(w[i] & 0x00F000F0u, odd, low);
    const uint32_t c = fma_f16x2(y & 0x000F000Fu, even, low), d = fma_f16x2(y & 0x00F000F0u, odd, low);
    const int chunk = (t & 1) * 4 + (i ^ (t & 2));
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(out + ((chunk ^ (row & 7)) * 16)), "r"(a), "r"(b), "r"(c),
                 "r"(d)
                 : "memory");
  }
}

__device__ __forceinline__ uint32_t twice_f16(float x) {
  const uint32_t h = __half_as_ushort(__float2half_rn(x));
  return h | h << 16;
}

__device__ __forceinline__ void unpack_role(const Int4AttnParams& p, Smem& sm, Cursor c, int64_t units, int warp, int lane) {
  const int g = lane >> 2, t = lane & 3;
  int v_exp = 0, v_exp_set = 0;
  int stage = 0;
  uint32_t raw_parity = 0;
  for (int64_t u = 0; u < units; ++u) {
    const int buf = static_cast<int>(u & 1);
    const uint32_t reuse = static_cast<uint32_t>(u >> 1);  // of the K buffer
    if (!wait_all(&sm.raw_full[stage], raw_parity, p.err)) return;
    // ---- the tile's largest magnitudes, over rows that are there (all warps alike)
    const uint32_t there = sm.raw_there[stage];
    const int pos0 = c.tile * kTile;
    float k_top = 0.f, v_top = 0.f;
    bool wild = false;  // a row that is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 32 * i + lane;
      const uint2 sc = sm.raw_scale[stage][row];
      const float ks = __uint_as_float(sc.x << 16), kl = __uint_as_float(sc.x & 0xFFFF0000u);
      const float vs = __uint_as_float(sc.y << 16), vl = __uint_as_float(sc.y & 0xFFFF0000u);
      const float kt = fmaxf(fabsf(kl), fabsf(fmaf(15.f, ks, kl))), vt = fmaxf(fabsf(vl), fabsf(fmaf(15.f, vs, vl)));
      const bool held = (there >> (row >> 4) & 1u) && pos0 + row < c.s.vis;
      if (held) {
        if (kt + fabsf(ks) + vt + fabsf(vs) < INFINITY) {  // a sum: NaN and infinity do not get lost
          k_top = fmaxf(k_top, kt);
          v_top = fmaxf(v_top, vt);
        } else {
          wild = true;
        }
      }
    }
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      k_top = fmaxf(k_top, __shfl_xor_sync(0xffffffffu, k_top, off));
      v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, off));
    }
    wild = __any_sync(0xffffffffu, wild);
    // largest magnitudes to between 2^-7 and 2^-6: steps times 2^24 stay below 2^16
    const int k_exp = k_top > 0.f ? max(-96, min(exponent(k_top), 110)) + 7 : 0;
    float change = 1.f;
    if (v_top > 0.f) {
      const int e = max(-96, min(exponent(v_top), 110)) + 7;
      if (!v_exp_set) {
        v_exp = e;
        v_exp_set = 1;
      } else if (e > v_exp) {
        change = v_exp - e < -126 ? 0.f : pow2(v_exp - e);
        v_exp = e;
      }
    }
    // ---- K
    if (reuse > 0 && !wait_all(&sm.k_free[buf], (reuse - 1) & 1u, p.err)) return;
    if (warp == 0 && lane == 0) {
      const int slot = static_cast<int>(u & 3);
      sm.k_back[slot] = pow2(k_exp);
      sm.v_change[slot] = change;
      sm.v_back[slot] = pow2(v_exp);
      sm.there[slot] = there | (wild ? kWild : 0u);
    }
    const float k_to = pow2(-k_exp), v_to = pow2(-v_exp);
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      if (half == 1 && u > 0 && !wait_all(&sm.v_free, static_cast<uint32_t>(u - 1) & 1u, p.err)) return;
      const uint32_t raw = smem_u32(half ? sm.raw_v[stage] : sm.raw_k[stage]);
      const uint32_t dst = smem_u32(half ? sm.v : sm.k[buf]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 32 * warp + 8 * i + g;
        const uint2 sc = sm.raw_scale[stage][row];
        const bool held = (there >> (row >> 4) & 1u) && pos0 + row < c.s.vis;
        const float ks = __uint_as_float(sc.x << 16), kl = __uint_as_float(sc.x & 0xFFFF0000u);
        const float vs = __uint_as_float(sc.y << 16), vl = __uint_as_float(sc.y & 0xFFFF0000u);
        const bool fine = fabsf(fmaf(15.f, ks, kl)) + fabsf(ks) + fabsf(fmaf(15.f, vs, vl)) + fabsf(vs) < INFINITY;
        float step = half ? vs * v_to : ks * k_to, low = half ? vl * v_to : kl * k_to;
        if (!held || !fine) {
          step = 0.f;
          low = held && half == 0 ? __uint_as_float(0x7FC00000u) : 0.f;
        }
        unpack_rows(raw, dst, row, t, twice_f16(step * 16777216.f), twice_f16(step * 1048576.f), twice_f16(low));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (half == 0) {
          mbar_arrive(&sm.k_full[buf]);
        } else {
          mbar_arrive(&sm.v_full);
          mbar_arrive(&sm.raw_empty[stage]);
        }
      }
    }
    if (++stage == kRaw) {
      stage = 0;
      raw_parity ^= 1u;
    }
    if (++c.tile == c.tiles && u + 1 < units) {
      next_pair(p, c);
      v_exp = v_exp_set = 0;
    }
  }
}

// ------------------------------------------------------------------------------------------ products
__device__ __forceinline__ void mma_role(const Int4AttnParams& p, Smem& sm, Cursor c, int64_t units) {
  const uint32_t idesc_s = tc::idesc_f16(128, 128, false, false), idesc_pv = tc::idesc_f16(128, 128, false, true);
  const uint32_t tmem = sm.tmem;
  uint64_t dq[2], dk[2];
  for (int i = 0; i < 2; ++i) {
    dq[i] = tc::smem_desc(smem_u32(sm.q[i]), 16, 1024, tc::kSw128);
    dk[i] = tc::smem_desc(smem_u32(sm.k[i]), 16, 1024, tc::kSw128);
  }
  const uint64_t dv = tc::smem_desc(smem_u32(sm.v), kOBytes, 1024, tc::kSw128);
  uint32_t q_parity = 0, p_parity[2] = {0, 0};
  bool ok = true;
  // O_g += P_g V, 16 positions at a time: V's rows are 128 bytes
  auto values = [&](int g, bool first) {
    ok = ok && wait_one(&sm.p_full[g], p_parity[g], p.err);
    p_parity[g] ^= 1u;
    if (!ok) return;
    tc::fence_after_sync();
#pragma unroll
    for (int i = 0; i < kTile / 16; ++i)
      tc::mma_f16_ts(tmem + 256 * g + 128, tmem + 256 * g + 8 * i, dv + static_cast<uint64_t>(i * (16 * 128 >> 4)), idesc_pv,
                     !first || i > 0 ? 1u : 0u);
  };
  for (int64_t u = 0; u < units && ok;) {
    const int n = static_cast<int>(min(units - u, static_cast<int64_t>(c.tiles - c.tile)));
    const int groups = c.s.nq * p.group - c.rg * kItem > kRows ? 2 : 1;
    for (int i = 0; i <= n && ok; ++i, ++u) {
      for (int g = 0; g < groups && ok; ++g) {
        if (i > 0) {
          if (g == 0) ok = wait_one(&sm.v_full, static_cast<uint32_t>(u - 1) & 1u, p.err);
          values(g, i == 1);
          if (ok && i == n) tc::commit(&sm.o_full[g]);
        }
        if (i < n && ok) {
          const int buf = static_cast<int>(u & 1);
          if (g == 0) ok = wait_one(&sm.k_full[buf], static_cast<uint32_t>(u >> 1) & 1u, p.err);
          if (i == 0) ok = ok && wait_one(&sm.q_full[g], q_parity >> g & 1u, p.err);
          if (!ok) break;
          tc::fence_after_sync();
#pragma unroll
          for (int k = 0; k < 8; ++k) {  // 16 values: 32 bytes, four to a block
            const uint64_t step = static_cast<uint64_t>((k >> 2) * (kOBytes >> 4) + (k & 3) * 2);
            mma_f16_ss(tmem + 256 * g, dq[g] + step, dk[buf] + step, idesc_s, k > 0 ? 1u : 0u);
          }
          tc::commit(&sm.s_full[g]);
        }
      }
      if (!ok) break;
      if (i > 0) tc::commit(&sm.v_free);
      if (i < n) tc::commit(&sm.k_free[u & 1]);
      if (i == n) --u;  // the loop's last step issued no scores
    }
    q_parity ^= groups == 2 ? 3u : 1u;
    c.tile += n;
    if (u < units) next_pair(p, c);
  }
  if (!ok) {  // products in flight must end before the CTA does
    tc::commit(&sm.drained);
    wait_one(&sm.drained, 0, p.err);
  }
}

// ------------------------------------------------------------------------------------------ softmax
// P of two scores: 2^(s cs + bias), and its part of the row's sum.
__device__ __forceinline__ void softmax_role(const Int4AttnParams& p, Smem& sm, Cursor c, int64_t units, int64_t ctas,
                                             int64_t total, int64_t u0, int g, int tid) {
  const int r = tid & 127, warp = r >> 5;
  const uint32_t s_tmem = sm.tmem + (static_cast<uint32_t>(32 * warp) << 16) + 256 * g, o_tmem = s_tmem + 128;
  uint32_t s_parity = 0, o_parity = 0;
  constexpr int kPart = kItem * (kHeadDim + 2);
  bool first_piece = true;
  for (int64_t u = 0; u < units;) {
    const int n = static_cast<int>(min(units - u, static_cast<int64_t>(c.tiles - c.tile)));
    const int rows = c.s.nq * p.group;
    if (rows - c.rg * kItem > g * kRows) {
      const int row = c.rg * kItem + g * kRows + r;
      const bool real = row < rows;
      const int token = row / p.group;
      const int64_t q_row = static_cast<int64_t>(c.s.q_first) + token;
      const int head = c.kvh * p.group + row - token * p.group;
      const int limit = real ? min(c.s.vis, token + c.s.nk - c.s.nq + 1) : c.s.vis;  // no row: zeros that see anything
      // ---- q: a power of two puts the largest value between 2^13 and 2^14
      float cs;
      {
        uint4 raw[16];
        const uint16_t* src = p.q + q_row * p.q_row_stride + head * kHeadDim;
#pragma unroll
        for (int i = 0; i < 16; ++i) raw[i] = real ? ldg_keep_v4(src + 8 * i) : make_uint4(0, 0, 0, 0);
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xFFFF0000u))));
        }
        const int e = amax > 0.f && amax < INFINITY ? max(-100, min(exponent(amax), 110)) - 13 : 0;
        const float to = p.scale_log2 < 0.f ? -pow2(-e) : pow2(-e);  // a negative scale turns q around
        cs = fabsf(p.scale_log2) * pow2(e);
#pragma unroll
        for (int i = 0; i < 16; ++i) {  // values 8 i .. 8 i + 7 in the order 0 4 1 5 2 6 3 7
          const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          float x[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[2 * k] = __uint_as_float(w[k] << 16) * to;
            x[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u) * to;
          }
          uint8_t* dst = sm.q[g] + (i >> 3) * kOBytes + r * 128 + (((i & 7) ^ (r & 7)) * 16);
          *reinterpret_cast<uint4*>(dst) = make_uint4(pack_f16x2(x[0], x[4]), pack_f16x2(x[1], x[5]),
                                                      pack_f16x2(x[2], x[6]), pack_f16x2(x[3], x[7]));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if ((tid & 31) == 0) mbar_arrive(&sm.q_full[g]);

      float m = kNone, l = 0.f, back = 1.f;
      for (int i = 0; i < n; ++i) {
        const int slot = static_cast<int>((u + i) & 3);
        // S_g of this tile done: so is O_g of the one before it
        if (!wait_all(&sm.s_full[g], s_parity, p.err)) return;
        s_parity ^= 1u;
        tc::fence_after_sync();
        const float ct = cs * sm.k_back[slot];
      back = sm.v_back[slot];
        const float change = sm.v_change[slot];
        const uint32_t there = sm.there[slot];
        const int seen = limit - (c.tile + i) * kTile;  // columns below this one
        // the polynomial would lose a NaN
        const bool full = __all_sync(0xffffffffu, there == 0xFFu && seen >= kTile);
        // ---- the row's maximum
        float top = kNone;
        uint32_t v[32];
        if (full) {
          float t0 = kNone, t1 = kNone, t2 = kNone, t3 = kNone;
#pragma unroll
          for (int c0 = 0; c0 < kTile; c0 += 32) {
            tmem_ld32(s_tmem + c0, v);
            tc::wait_ld();
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              t0 = fmaxf(t0, fmaxf(__uint_as_float(v[k]), __uint_as_float(v[k + 1])));
              t1 = fmaxf(t1, fmaxf(__uint_as_float(v[k + 2]), __uint_as_float(v[k + 3])));
              t2 = fmaxf(t2, fmaxf(__uint_as_float(v[k + 4]), __uint_as_float(v[k + 5])));
              t3 = fmaxf(t3, fmaxf(__uint_as_float(v[k + 6]), __uint_as_float(v[k + 7])));
            }
          }
          top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
        } else {
#pragma unroll 1
          for (int c0 = 0; c0 < kTile; c0 += 32) {
            tmem_ld32(s_tmem + c0, v);
            tc::wait_ld();
            const uint32_t part = there >> (c0 >> 4);
            const uint32_t held = ((part & 1u) ? 0xFFFFu : 0u) | ((part & 2u) ? 0xFFFF0000u : 0u);
            const int left = seen - c0;
            const uint32_t mask = held & (left >= 32 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << left) - 1u);
#pragma unroll
            for (int k = 0; k < 32; ++k) top = fmaxf(top, mask >> k & 1u ? __uint_as_float(v[k]) : kNone);
          }
        }
        top = top == kNone ? kNone : top * ct;  // ct is not negative
        // ---- a new reference maximum where it lags too far, and V's power of two
        float f = change;
        if (top > m + kSlack) {
          const float lag = ex2(m - top);
          m = top;
          l *= lag;
          f *= lag;
        }
        if (i > 0 && __any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll 1
          for (int c0 = 0; c0 < kHeadDim; c0 += 32) {
            tmem_ld32(o_tmem + c0, v);
            tc::wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
            tmem_st32(o_tmem + c0, v);
          }
          tc::wait_st();
        }
        // ---- P over the columns of S that have been read
        const float bias = kLift - m;
        uint64_t sum0 = f2_pack(0.f, 0.f), sum1 = sum0;
        const uint64_t ct2 = f2_pack(ct, ct), bias2 = f2_pack(bias, bias);
        if (full) {
#pragma unroll 1
          for (int c0 = 0; c0 < kTile; c0 += 32) {
            tmem_ld32(s_tmem + c0, v);
            tc::wait_ld();
            uint32_t pw[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const uint64_t x = f2_fma(f2_pack(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), ct2, bias2);
              float x0, x1, p0, p1;
              f2_unpack(x, x0, x1);
              if (k % 3 == 2) {
                exp2_poly_x2(x0, x1, p0, p1);
              } else {
                p0 = ex2(x0);
                p1 = ex2(x1);
              }
              if (k & 1) {
                sum1 = f2_add(sum1, f2_pack(p0, p1));
              } else {
                sum0 = f2_add(sum0, f2_pack(p0, p1));
              }
              pw[k] = pack_f16x2(p0, p1);
            }
            tc::st16u(s_tmem + c0 / 2, pw);
          }
        } else {
#pragma unroll 1
          for (int c0 = 0; c0 < kTile; c0 += 32) {
            tmem_ld32(s_tmem + c0, v);
            tc::wait_ld();
            const uint32_t part = there >> (c0 >> 4);
            const uint32_t held = ((part & 1u) ? 0xFFFFu : 0u) | ((part & 2u) ? 0xFFFF0000u : 0u);
            const int left = seen - c0;
            const uint32_t mask = held & (left >= 32 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << left) - 1u);
            uint32_t pw[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float p0 = mask >> (2 * k) & 1u ? ex2(fmaf(__uint_as_float(v[2 * k]), ct, bias)) : 0.f;
              const float p1 = mask >> (2 * k + 1) & 1u ? ex2(fmaf(__uint_as_float(v[2 * k + 1]), ct, bias)) : 0.f;
              sum0 = f2_add(sum0, f2_pack(p0, p1));
              pw[k] = pack_f16x2(p0, p1);
            }
            tc::st16u(s_tmem + c0 / 2, pw);
          }
        }
        float a0, a1, b0, b1;
        f2_unpack(sum0, a0, a1);
        f2_unpack(sum1, b0, b1);
        l += (a0 + a1) + (b0 + b1);
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if ((tid & 31) == 0) mbar_arrive(&sm.p_full[g]);
      }
      // ---- the piece's end
      if (!wait_all(&sm.o_full[g], o_parity, p.err)) return;
      o_parity ^= 1u;
      tc::fence_after_sync();
      const bool whole = c.tile == 0 && n == c.tiles;
      const float f = !whole ? back : l == 0.f ? 0.f : __fdiv_rn(back, l);
      float* part = p.partials + (2 * static_cast<int64_t>(blockIdx.x) + (first_piece ? 0 : 1)) * kPart +
                    (g * kRows + r) * kHeadDim;
      uint16_t* dst = p.out + q_row * p.out_row_stride + head * kHeadDim;
#pragma unroll 1
      for (int c0 = 0; c0 < kHeadDim; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(o_tmem + c0, v);
        tc::wait_ld();
#pragma unroll
        for (int k = 0; k < 32; k += 8) {  // back from the order 0 4 1 5 2 6 3 7
          const float y[8] = {__uint_as_float(v[k]) * f,     __uint_as_float(v[k + 2]) * f, __uint_as_float(v[k + 4]) * f,
                              __uint_as_float(v[k + 6]) * f, __uint_as_float(v[k + 1]) * f, __uint_as_float(v[k + 3]) * f,
                              __uint_as_float(v[k + 5]) * f, __uint_as_float(v[k + 7]) * f};
          if (!whole) {
            *reinterpret_cast<float4*>(part + c0 + k) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4*>(part + c0 + k + 4) = make_float4(y[4], y[5], y[6], y[7]);
          } else if (real) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(y[2 * j], y[2 * j + 1]);
              w[j] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(dst + c0 + k) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (!whole)
        *reinterpret_cast<float2*>(p.partials + (2 * static_cast<int64_t>(blockIdx.x) + (first_piece ? 0 : 1)) * kPart +
                                   kItem * kHeadDim + 2 * (g * kRows + r)) = make_float2(m, l);
      tc::fence_before_sync();  // O has been read before the next piece's first P is announced
    }
    u += n;
    if (u < units) {
      c.tile += n;
      next_pair(p, c);
    } else if (tid == 0) {  // group 0 always has rows
      Cut cut = {};
      if (c.tile == 0 && n < c.tiles) {
        cut.parts = static_cast<int>(owner(u0 + u - n + c.tiles - 1, ctas, total) - blockIdx.x + 1);
        cut.slot = 2 * blockIdx.x + (first_piece ? 0 : 1);
        cut.rows = min(kItem, rows - c.rg * kItem);
        cut.first_row = c.rg * kItem;
        cut.token = c.s.q_first;
        cut.head = c.kvh * p.group;
      }
      reinterpret_cast<Cut*>(p.cuts)[blockIdx.x] = cut;
    }
    first_piece = false;
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
      mbar_init(&sm.q_full[i], 4);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.o_full[i], 1);
    }
    mbar_init(&sm.v_full, 4);
    mbar_init(&sm.v_free, 1);
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
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);
  if (blockIdx.x >= ctas) {
    if (tid == 0) reinterpret_cast<Cut*>(p.cuts)[blockIdx.x].parts = 0;
    return;
  }
  const int64_t u0 = range_begin(blockIdx.x, ctas, total), units = range_begin(blockIdx.x + 1, ctas, total) - u0;
  if (before <= u0 && u0 < before + mine) {
    int64_t at = before;
    int s = s0;
    for (; s < s1; ++s) {
      const int64_t n = units_of(p, seq_of(p, s));
      if (u0 < at + n) break;
      at += n;
    }
    sm.first_seq = s;
    sm.first_unit = at;
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
    int64_t rest = u0 - sm.first_unit;
    for (c.rg = 0;; ++c.rg) {
      c.tiles = tiles_of(p, c.s, c.rg);
      if (rest < static_cast<int64_t>(c.tiles) * p.num_kv_heads) break;
      rest -= static_cast<int64_t>(c.tiles) * p.num_kv_heads;
    }
    c.kvh = static_cast<int>(rest / c.tiles);
    c.tile = static_cast<int>(rest - static_cast<int64_t>(c.kvh) * c.tiles);
  }

  if (warp < kUnpackWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    softmax_role(p, sm, c, units, ctas, total, u0, warp >> 2, tid);
  } else if (warp < kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUnpackRegs));
    unpack_role(p, sm, c, units, warp - kUnpackWarp, lane);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kLoadWarp) {
      load_role(p, map_k, map_v, sm, c, units, lane);
    } else if (warp == kMmaWarp && lane == 0) {
      mma_role(p, sm, c, units);
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

int64_t int4_prefill_workspace_bytes(int num_sms) {
  return static_cast<int64_t>(num_sms) * (sizeof(Cut) + 2ll * kItem * (kHeadDim + 2) * 4);
}

cudaError_t launch_int4_prefill(Int4AttnParams p, const CUtensorMap& map_k, const CUtensorMap& map_v, void* workspace,
                                int num_sms, cudaStream_t stream) {
  p.cuts = workspace;
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + num_sms * sizeof(Cut));
  p.unit_pages = kTile / p.block_size;
  p.unit_rest = kTile % p.block_size;
  cudaError_t e = cudaFuncSetAttribute(int4_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return e;
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
  e = cudaLaunchKernelEx(&cfg, int4_prefill_kernel, p, map_k, map_v);
  if (e != cudaSuccess || num_sms < 2) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(num_sms - 1), 16);
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, int4_join_kernel<kItem>, p);
}

}  // namespace fp8attn
