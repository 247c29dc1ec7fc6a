// Tree attention over the paged cache for more than 16 query rows per KV head,
// on the 5th-gen tensor cores (tcgen05 + TMEM): bf16 queries, bf16 / int8 / e4m3
// cache, head_dim a multiple of 16.
//
//   S [128 rows, 128 keys] = Q K^T    (SS MMA, both K-major)
//   O [128 rows, d]       += P V      (TS MMA: P over S in TMEM; V MN-major)
// A CTA walks over its span of key tiles (tree_attention.cuh) with two streams,
// each with its own S / P, O, running max and sums, so that the softmax of one
// runs beside the MMAs of the other:
//   one tile of queries (128 rows)   stream = key tile mod 2, added up at the end
//                                    of a piece
//   two tiles (256 rows, beside 8-bit codes only)   one a stream; every key tile is
//                                    loaded and widened once for both
// Roles, one warp or group of warps each:
//   8 warps      softmax, thread = query row (TMEM lane); they bring in the
//                queries of a piece and write its results
//   1 warp       TMEM owner and MMA issuer; clears bf16 value rows that do not exist
//   2 warps      page lookups and copies, one K (and the scales), one V: the rings
//                of tiles stay full.  bf16 tiles come as TMA boxes of up to 128
//                rows of a page straight into the layout of the MMA, 8-bit codes as
//                bulk copies of rows that are neighbours in the page
//   8 warps      (8-bit) widen codes to fp16, exactly, one group K, the other V.
//                A warp reads the codes of its 32 rows of the tile into registers
//                from the place where it then writes their values.  Scales act
//                on S and P in fp32; the queries are held in fp16 too, each row
//                scaled by a power of two that takes its largest element to 2^14:
//                bf16 digits fit, and what falls below fp16's range is under
//                2^-39 of that element
// K and V have rings of their own, so that neither copy waits behind the other
// and every role sees every use of the barriers that it waits on.
// The running max of a row moves (with O and the sums rescaled) only when a
// score passes it by 2^8.  P is rounded once for its MMA, to bf16 beside bf16
// values (a relative 2^-8 of each weight) and to fp16 beside 8-bit ones (2^-11):
// there P carries the V scale, so the max is taken over score + log2(scale), in
// units that keep P below 2^14 (kWeightUp in tree_attention.cuh; below 2^-20 of
// the largest fp16 is subnormal and holds P to 2^-31 of that).
//
// Measured (8 KV heads of 128, 4 query heads each): 64 tokens over 131072, bf16,
// 182 us or 756 TFLOP/s; int8, 292 us; 13 tokens of 16 sequences over 4001, int8,
// 96 us; bf16 73 us.  Neither memory nor tensor cores are full: what bounds it
// is the chain scores -> weights -> values -> next scores of a stream (its scores
// and weights share TMEM) and the instruction cache, which all roles share.
//
// Waits are bounded (2 s).  After one has run out a role sets the error word
// and walks through the rest of its loop without waiting; the outputs are then
// invalid.  Named barriers still match -- whether a warp comes to one depends on
// lengths and arguments alone, never on what another role left in shared
// memory --, the copy warps begin no copy into a place whose last one has not
// landed and wait for all of theirs, and TMEM is freed.
#include <string>
#include <type_traits>

#include "tc05.cuh"
#include "tree_attention.cuh"

namespace dcc {

using namespace tc05;

int attn_error_flag_address(unsigned int** out);
unsigned int* attn_error_report();

namespace tt {

constexpr int kRing = 8;  // scales and masks of the last K tiles
constexpr int kFetch = 4;   // K tiles between a page lookup and its use
constexpr size_t kSmemLimit = 232448;

template <int kMode, int kD, bool kPair>  // cache format, padded head_dim, two tiles of queries
struct Shape {
  static constexpr bool k8 = kMode == DCC_KV_INT8 || kMode == DCC_KV_E4M3;
  static constexpr int kRows = kPair ? 256 : 128;
  static constexpr int kTile = 128 * kD * 2;          // Q, K or V tile of 16-bit values
  static constexpr int kBlocks = kD / 64;             // 64-column blocks of 128 swizzled rows
  static constexpr uint32_t kColS = 0, kColO = 256;   // TMEM columns, 128 a stream
  static constexpr int kArrays = k8 ? 3 : 1;          // bias; K and V scales
  static constexpr size_t kFixed = (size_t)kRows * kD * 2 + (size_t)kRing * kArrays * 512 + 2 * 4 * 512 + 3 * 1024 + kRows * 4 + 40;
  static constexpr int kFit = (int)((kSmemLimit - kFixed) / kTile);
  static constexpr int kSlotsV = (kFit + 1) / 2 < 4 ? (kFit + 1) / 2 : 4, kSlotsK = kFit / 2 < 4 ? kFit / 2 : 4;
  static constexpr int kSlots = kSlotsK + kSlotsV;
  static_assert(kSlotsK >= 2, "rings");
  // K tile j + kRing is copied once K tile j + kRing - kSlotsK has been consumed,
  // and those scores were issued behind the product of the tile two before: that
  // has to be tile j or a later one, so that nobody reads its scales any more
  static_assert(kRing - kSlotsK - 2 >= 0, "ring of scales");
  static constexpr int kWiden = k8 ? 8 : 0;
  static constexpr int kGroups = 3 + kWiden / 4;      // warpgroups
  static constexpr int kThreads = kGroups * 128;
  static constexpr int kRegsLaunch = 65536 / kThreads / 8 * 8;
  static constexpr int kRegsSoftmax = k8 ? 136 : 192;
  static constexpr int kRegsWork = k8 ? 88 : 112;     // issuer, copies
  static constexpr int kRegsWiden = 56;
  static_assert(2 * kRegsSoftmax + kRegsWork + kWiden / 4 * kRegsWiden <= kGroups * kRegsLaunch, "register split");
  static_assert(kRegsWork <= kRegsLaunch && kRegsWiden <= kRegsLaunch && kRegsSoftmax >= kRegsLaunch, "register split");
};

template <typename X>
struct Smem {
  unsigned char slot[X::kSlots][X::kTile];
  unsigned char q[X::kRows / 128][X::kTile];
  __align__(16) float side[kRing][X::kArrays][128];  // bias, k_scale, v_scale
  // of a stream's tile: bias in powers of two (-inf: hidden), K scale, V scale, the
  // V scale's logarithm with the bias
  __align__(16) float bias[2][128];
  __align__(16) float ks[2][128], vs[2][128], lift[2][128];
  float most[2][4];                                   // largest V scale of a stream's first tile, by warp
  int up[2];                                          // its exponent (see kWeightUp)
  __align__(16) uint8_t vis[kRing][16];               // bits: keys that exist
  int32_t pages[2][kFetch][16];                       // of every eighth key of the next K and V tiles
  float qf[X::kRows];                                 // what undoes the scaling of a query row
  union {
    float2 ml[2][128];                                // max and sum of a row, to add the streams up
    TreePlanSmem plan;                                // only before the roles begin
  };
  TreePlan span;
  uint64_t bar_raw[X::kSlots], bar_full[X::kSlots], bar_empty[X::kSlots], bar_side[kRing], bar_q, bar_s[2], bar_p[2],
      bar_o[2], bar_end;
  uint32_t tmem;
};
template <int kMode, int kD, bool kPair>
using SmemOf = Smem<Shape<kMode, kD, kPair>>;

// Waits with a hint to sleep, so that idle roles leave the issue slots to the
// others; gives up after 2 s.
__device__ __forceinline__ bool sleep_wait(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(100000u)
        : "memory");
    if (ok) return true;
    if (global_ns() - t0 > 2000000000ull) return false;
  }
}
__device__ __forceinline__ bool wait_all_lanes(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, sleep_wait(bar, parity)) != 0;
}
// A wait that is skipped once one has run out.
__device__ __forceinline__ void wait_or_skip(bool& ok, uint64_t* bar, uint32_t parity) {
  if (ok) ok = wait_all_lanes(bar, parity);
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 3, 256;\n" ::: "memory"); }
__device__ __forceinline__ void group_sync(int wg) { asm volatile("bar.sync %0, 128;\n" ::"r"(1 + wg) : "memory"); }
__device__ __forceinline__ void copy_async_word(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
// Arrives (counted beforehand) once this thread's cp.async so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// A place of the ring and the parity of its current use.
struct Place {
  int slots, slot = 0;
  uint32_t use = 0;
  __device__ __forceinline__ explicit Place(int n) : slots(n) {}
  __device__ __forceinline__ void next() {
    if (++slot == slots) {
      slot = 0;
      use ^= 1;
    }
  }
};

// The tiles of a CTA, one after the other over its row tiles and pieces.
struct Tiles {
  TreeWalk walk;
  TreePiece w;
  int rt, kt;
  bool first, last;  // of its piece
  __device__ __forceinline__ void start(const TreeParams& p, const TreePlan& pl) {
    rt = blockIdx.x % p.n_groups;
    walk.start(p, pl);
    kt = 0;
    w.k1 = 0;
  }
  __device__ __forceinline__ void next(const TreeParams& p, const TreePlan& pl) {
    first = false;
    if (++kt >= w.k1) {
      if (!walk.next(p, w)) {
        rt += p.n_groups;
        walk.start(p, pl);
        walk.next(p, w);
      }
      kt = w.k0;
      first = true;
    }
    last = kt + 1 == w.k1;
  }
};

struct TreeMaps {
  CUtensorMap k, v;  // bf16 rows of the pools
  int page_rows;     // the largest power of two up to 128 that divides page_size, at least 8
};

// Descriptor of a 128-byte swizzled operand: the address changes, the rest is
// fixed (see sdesc_sw128).
__device__ __forceinline__ uint64_t desc_at(uint32_t saddr, uint32_t lbo) {
  const uint32_t lo = (saddr >> 4) | (lbo >> 4) << 16;
  return (uint64_t)lo | (uint64_t)((1024u >> 4) | 1u << 14 | 2u << 29) << 32;
}

// ---- copies ----------------------------------------------------------------------------
// One code for K and V, as in the widening: all roles together just fit into the
// instruction cache (an instance for each: 111 instead of 102 us for 16
// sequences of 13 tokens over 4k int8 tokens; the softmax below, unrolled over all
// 128 keys instead of 32: 185 instead of 129 us).
template <int kMode, int kD, bool kPair>
__device__ __forceinline__ void copies(const TreeParams& p, const TreeMaps& maps, SmemOf<kMode, kD, kPair>& sm, bool is_v, int n,
                                       int lane, bool& ok) {
  using X = Shape<kMode, kD, kPair>;
  const int first_slot = is_v ? X::kSlotsK : 0;
  const TreePlan& pl = sm.span;
  const uint32_t row_bytes = (uint32_t)p.c.head_dim * (X::k8 ? 1 : 2);
  const bool pow2 = (p.c.page_size & (p.c.page_size - 1)) == 0;
  const int shift = 31 - __clz(p.c.page_size);
  // rows of a copy: 8-bit rows shorter than their 128-byte place come in eights,
  // so that a warp's rows land within its own part of the tile
  const int rows = X::k8 && p.c.head_dim != 128 ? 8 : maps.page_rows;
  const bool leader = lane < 16 && ((8 * lane) & (rows - 1)) == 0;
  const uint32_t bytes = (uint32_t)rows * (X::k8 ? row_bytes : X::kBlocks * 128);
  const uint32_t slot0 = smem_u32(sm.slot[first_slot]) + (uint32_t)lane * 1024;
  const int page_step = p.c.n_kv_heads * p.c.page_size;
  Tiles t;
  t.start(p, pl);
  // lane < 16: rows 8 lane .. 8 lane + 7 of a tile (a page holds all eight or
  // none).  Their page numbers are on their way to shared memory kFetch tiles
  // ahead -- a register that waits for a load would stall the warp when the
  // queue moves on --, the row in the page and the rows that exist are known
  int add[kFetch], left[kFetch];
  int fetched = 0;
  auto fetch = [&]() {
    left[kFetch - 1] = 0;
    if (fetched < n) {
      t.next(p, pl);
      const int pos = t.kt * kTreeKeys + 8 * lane;
      left[kFetch - 1] = lane < 16 ? (int)(t.w.s.total - pos) : 0;
      if (left[kFetch - 1] > 0) {
        const int s = pow2 ? pos >> shift : pos / p.c.page_size;
        add[kFetch - 1] = t.w.hk * p.c.page_size + pos - s * p.c.page_size;
        copy_async_word(smem_u32(&sm.pages[is_v][fetched % kFetch][lane]), p.q.page_table + (int64_t)t.w.b * p.q.table_stride + s);
      }
      ++fetched;
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  auto shift_down = [&]() {
#pragma unroll
    for (int f = 0; f + 1 < kFetch; ++f) {
      add[f] = add[f + 1];
      left[f] = left[f + 1];
    }
  };
#pragma unroll 1
  for (int i = 0; i < kFetch; ++i) {
    shift_down();
    fetch();
  }
  Place at(is_v ? X::kSlotsV : X::kSlotsK);
  int j = 0;
#pragma unroll 1
  for (; j < n; ++j) {
    const int slot = first_slot + at.slot;
    uint64_t* bar = X::k8 ? &sm.bar_raw[slot] : &sm.bar_full[slot];
    if (j >= at.slots) {
      wait_or_skip(ok, &sm.bar_empty[slot], at.use ^ 1);
      wait_or_skip(ok, bar, at.use ^ 1);  // the copies of before have landed, also if others gave up and passed the tile on
      if (!ok) break;
    }
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kFetch - 1) : "memory");  // this lane's own page number
    int row = -1;
    if (left[0] > 0) {
      const int page = sm.pages[is_v][j % kFetch][lane];
      if (page >= 0 && page < p.c.n_pages) row = page * page_step + add[0];
    }
    if (!is_v) {
      const int ring = j % kRing;
      if (lane < 16) sm.vis[ring][lane] = row >= 0 ? (uint8_t)(left[0] >= 8 ? 0xff : (1 << left[0]) - 1) : (uint8_t)0;
      __syncwarp();  // vis before the arrival
      if (lane == 0) mbar_arrive(&sm.bar_side[ring]);
      if (X::k8 || p.c.bias) {  // of four keys a lane
        const int eight = __shfl_sync(0xffffffffu, row, lane >> 1);
        const uint32_t to = smem_u32(&sm.side[ring][0][4 * lane]), size = eight >= 0 ? 16 : 0;
        const int from = eight >= 0 ? eight + 4 * (lane & 1) : 0;
        if (p.c.bias) copy_async(to, p.c.bias + from, size);
        if constexpr (X::k8) {
          copy_async(to + 512, p.c.k_scale + from, size);
          copy_async(to + 1024, p.c.v_scale + from, size);
        }
        cp_async_arrive(&sm.bar_side[ring]);
      }
    }
    const bool lead = row >= 0 && leader;
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, lead));
    if (lane == 0) mbar_expect_tx(bar, count * bytes);
    __syncwarp();
    if (lead) {
      const uint32_t dst = slot0 + (uint32_t)at.slot * X::kTile;
      if constexpr (X::k8) {
        bulk_load(dst, static_cast<const unsigned char*>(is_v ? p.c.v : p.c.k) + (int64_t)row * row_bytes, bytes, bar);
      } else {
#pragma unroll
        for (int b = 0; b < X::kBlocks; ++b) tma_load_2d(dst + b * 16384, is_v ? &maps.v : &maps.k, bar, 64 * b, row);
      }
    }
    shift_down();
    fetch();
    at.next();
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");
  // nothing may still be on its way into shared memory when the CTA ends
  for (int i = 0; i < min(j, at.slots); ++i) {
    const uint32_t last = (uint32_t)((j - 1 - i) / at.slots);  // use of slot i
    if (!wait_all_lanes(X::k8 ? &sm.bar_raw[first_slot + i] : &sm.bar_full[first_slot + i], last & 1)) ok = false;
  }
}

// ---- 8-bit: codes to values ----------------------------------------------------------------
// Warps w = 0 .. 3 of the group for K or for V.
template <int kMode, int kD, bool kPair>
__device__ __forceinline__ void widen_tiles(const TreeParams& p, SmemOf<kMode, kD, kPair>& sm, bool is_v, int n, int w, int lane,
                                            bool& ok) {
  using X = Shape<kMode, kD, kPair>;
  constexpr int kPerRow = kD / 16;                  // 16-byte chunks of codes in a row
  constexpr int kRowsPer = 32 / kPerRow;            // rows of one step of the warp: 4 or 8
  constexpr int kTurn = 8 / kRowsPer;               // steps until the pattern of rows repeats, 1024 bytes on
  // lane -> (chunk, row of the step): eight lanes in a row write the eight
  // 16-byte banks of two rows, whose value chunks are two apart
  const int chunk = kPerRow == 8 ? (lane & 3) | ((lane >> 1) & 4) : lane & 3;
  const int sub = kPerRow == 8 ? ((lane >> 2) & 1) | ((lane >> 3) & 2) : lane >> 2;
  const bool chunk_real = chunk * 16 < p.c.head_dim;
  // offsets in a tile: codes, value chunks 2 chunk and 2 chunk + 1 (128-byte rows
  // of a 64-column block, chunks xor-ed with the row)
  uint32_t from[kTurn], to[kTurn][2];
#pragma unroll
  for (int i = 0; i < kTurn; ++i) {
    const int r = 32 * w + i * kRowsPer + sub;
    from[i] = (uint32_t)((r >> 3) * 1024 + (r & 7) * p.c.head_dim + chunk * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 2 * chunk + h;
      to[i][h] = (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    }
  }
  const int first_slot = is_v ? X::kSlotsK : 0;
  Place at(is_v ? X::kSlotsV : X::kSlotsK);
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const int slot = first_slot + at.slot;
    wait_or_skip(ok, &sm.bar_raw[slot], at.use);
    const uint32_t tile = smem_u32(sm.slot[slot]);
    // whatever the slot held in rows that do not exist may be a NaN in e4m3,
    // which a zero weight would not hide
    uint32_t real = 0xffffffffu;
    if (kMode == DCC_KV_E4M3 && is_v) {
      wait_or_skip(ok, &sm.bar_side[j % kRing], (uint32_t)(j / kRing) & 1);
      real = *reinterpret_cast<const uint32_t*>(&sm.vis[j % kRing][4 * w]) >> sub;
    }
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {  // 16 rows at a time
      uint4 raw[2 * kTurn];
#pragma unroll
      for (int s = 0; s < 2 * kTurn; ++s)
        raw[s] = chunk_real && (kMode != DCC_KV_E4M3 || ((real >> (8 * (s / kTurn + 2 * half) + s % kTurn * kRowsPer)) & 1))
                     ? ld_shared_v4(tile + from[s % kTurn] + (s / kTurn + 2 * half) * 1024)
                     : make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();  // this warp alone reads and writes these rows
#pragma unroll
      for (int s = 0; s < 2 * kTurn; ++s) {
        uint32_t h[8];
        widen_word<kMode>(raw[s].x, h[0], h[1]);
        widen_word<kMode>(raw[s].y, h[2], h[3]);
        widen_word<kMode>(raw[s].z, h[4], h[5]);
        widen_word<kMode>(raw[s].w, h[6], h[7]);
        const uint32_t on = (s / kTurn + 2 * half) * 1024;
        st_shared_v4(tile + to[s % kTurn][0] + on, h[0], h[1], h[2], h[3]);
        st_shared_v4(tile + to[s % kTurn][1] + on, h[4], h[5], h[6], h[7]);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.bar_full[slot]);
    at.next();
  }
}

// One lane, the same every time; with it and a warp index that is the same in all
// lanes the operands of MMAs stay in uniform registers.
__device__ __forceinline__ bool elected() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e != 0;
}
// ---- MMA issuer ----------------------------------------------------------------------
// bf16 value rows that do not exist hold whatever the page or the slot held,
// and newest values that are not finite must not reach rows that do not see
// them (0 * inf): both become zeros here; the softmax marks the rows that do
// see the latter.  (int8 codes are always finite; e4m3 has a NaN code, which a
// pool may hold that was filled elsewhere.)
template <int kMode, int kD, bool kPair>
__device__ __forceinline__ void clear_values(SmemOf<kMode, kD, kPair>& sm, uint32_t tile, int ring, bool newest, int64_t first,
                                             int lane) {
  constexpr int kPerRow = kD / 8, kRowsPer = 32 / kPerRow;
  constexpr uint32_t kTop = kMode == DCC_KV_BF16 ? 0x7f80u : 0x7c00u;  // exponent of what is not finite, bf16 and fp16
  const int chunk = lane % kPerRow, sub = lane / kPerRow;
#pragma unroll 1
  for (int r = sub; r < kTreeKeys; r += kRowsPer) {
    const bool exists = (sm.vis[ring][r >> 3] >> (r & 7)) & 1;
    if (exists && !(newest && first + r >= 0)) continue;
    const uint32_t a = tile + (uint32_t)((chunk >> 3) * 16384 + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
    uint32_t u[4] = {0u, 0u, 0u, 0u};
    if (exists) {
      const uint4 v = ld_shared_v4(a);
      u[0] = v.x, u[1] = v.y, u[2] = v.z, u[3] = v.w;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if ((u[c] & kTop) == kTop) u[c] &= 0xffff0000u;
        if ((u[c] & kTop << 16) == kTop << 16) u[c] &= 0x0000ffffu;
      }
    }
    st_shared_v4(a, u[0], u[1], u[2], u[3]);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

template <int kMode, int kD, bool kPair>
__device__ __forceinline__ void issuer(const TreeParams& p, SmemOf<kMode, kD, kPair>& sm, int n, bool guard, uint32_t tm, int lane,
                                       bool& ok) {
  using X = Shape<kMode, kD, kPair>;
  const uint32_t id_s = X::k8 ? idesc_f16_f32(128, 128, 0, 0) : idesc_bf16_f32(128, 128, 0, 0);
  const uint32_t id_o = X::k8 ? idesc_f16_f32(128, kD, 0, 1) : idesc_bf16_f32(128, kD, 0, 1);
  const uint64_t q0 = desc_at(smem_u32(sm.q[0]), 16);
  const uint32_t k0 = smem_u32(sm.slot[0]), v0 = smem_u32(sm.slot[X::kSlotsK]);
  Tiles ts, tv;  // of the next scores, of the next values
  ts.start(p, sm.span);
  tv.start(p, sm.span);
  Place at_k(X::kSlotsK), at_v(X::kSlotsV);
  uint32_t pieces = 0;
  auto scores = [&](int stream, uint64_t q, uint64_t k) {
    if (elected()) {
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk)
        umma_ss(tm + X::kColS + (uint32_t)stream * 128, q + ((kk >> 2) * 16384 + (kk & 3) * 32) / 16,
                k + ((kk >> 2) * 16384 + (kk & 3) * 32) / 16, id_s, kk > 0);
      umma_commit(&sm.bar_s[stream]);
    }
    __syncwarp();
  };
  // the K tile of `ts` is there, and the queries of its piece
  auto this_k = [&]() {
    if (ts.first) {
      wait_or_skip(ok, &sm.bar_q, pieces & 1);
      ++pieces;
    }
    wait_or_skip(ok, &sm.bar_full[at_k.slot], at_k.use);
    tc_fence_after();
    return desc_at(k0 + (uint32_t)at_k.slot * X::kTile, 16);
  };
  auto done_k = [&]() {
    if (elected()) umma_commit(&sm.bar_empty[at_k.slot]);
    __syncwarp();
    at_k.next();
  };
  auto next_v = [&](int j) {
    tv.next(p, sm.span);
    wait_or_skip(ok, &sm.bar_full[X::kSlotsK + at_v.slot], at_v.use);
    const uint32_t tile = v0 + (uint32_t)at_v.slot * X::kTile;
    if constexpr (kMode != DCC_KV_INT8) {
      const int ring = j % kRing;
      wait_or_skip(ok, &sm.bar_side[ring], (uint32_t)(j / kRing) & 1);
      const uint4 vis = *reinterpret_cast<const uint4*>(sm.vis[ring]);
      const int64_t first = (int64_t)tv.kt * kTreeKeys - tv.w.s.ctx;  // of the tile, behind the context
      const bool newest = guard && first + kTreeKeys > 0;
      if ((!X::k8 && (vis.x & vis.y & vis.z & vis.w) != 0xffffffffu) || newest)
        clear_values<kMode, kD, kPair>(sm, tile, ring, newest, first, lane);
    }
    return desc_at(tile, 16384);
  };
  auto values = [&](int stream, uint64_t v, bool first) {
    tc_fence_after();
    if (elected()) {
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        umma_ts(tm + X::kColO + (uint32_t)stream * 128, tm + X::kColS + (uint32_t)stream * 128 + kk * 8, v + kk * 128, id_o,
                (first && kk == 0) ? 0u : 1u);
      umma_commit(&sm.bar_o[stream]);
    }
    __syncwarp();
  };
  auto done_v = [&]() {
    if (elected()) umma_commit(&sm.bar_empty[X::kSlotsK + at_v.slot]);
    __syncwarp();
    at_v.next();
  };
  // A stream's next scores overwrite its last weights: they are issued behind
  // the product that reads those, and MMAs of one thread run in order.
  if constexpr (kPair) {
    ts.next(p, sm.span);
    uint64_t k = this_k();
    scores(0, q0, k);
    scores(1, q0 + X::kTile / 16, k);
    done_k();
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const uint64_t v = next_v(j);
      const bool first = tv.first, more = j + 1 < n;
      wait_or_skip(ok, &sm.bar_p[0], (uint32_t)j & 1);
      values(0, v, first);
      // with a new piece the queries change: only behind both streams' products
      if (more && !tv.last) {
        ts.next(p, sm.span);
        k = this_k();
        scores(0, q0, k);
      }
      wait_or_skip(ok, &sm.bar_p[1], (uint32_t)j & 1);
      values(1, v, first);
      done_v();
      if (more) {
        if (tv.last) {
          ts.next(p, sm.span);
          k = this_k();
          scores(0, q0, k);
        }
        scores(1, q0 + X::kTile / 16, k);
        done_k();
      }
    }
  } else {
    // scores run two tiles ahead of the products, but those of a new piece only
    // start behind all products of the one before, whose end its queries wait for
    int js = 0;
    ts.next(p, sm.span);
    auto feed = [&](int done) {
      while (js < n && js < done + 2 && (!ts.first || js == done)) {
        scores(js & 1, q0, this_k());
        done_k();
        if (++js < n) ts.next(p, sm.span);
      }
    };
    feed(0);
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const uint64_t v = next_v(j);
      const bool first = tv.kt - tv.w.k0 < 2;  // of the stream in this piece
      wait_or_skip(ok, &sm.bar_p[j & 1], (uint32_t)(j >> 1) & 1);
      values(j & 1, v, first);
      done_v();
      feed(j + 1);
    }
  }
  // every MMA has finished before TMEM is freed, also after a wait that ran out
  if (elected()) umma_commit(&sm.bar_end);
  __syncwarp();
  if (!wait_all_lanes(&sm.bar_end, 0)) ok = false;
}

// ---- softmax and results --------------------------------------------------------------
template <int kMode, int kD, bool kPair>
__device__ __forceinline__ void softmax(const TreeParams& p, SmemOf<kMode, kD, kPair>& sm, bool guard, int span, uint32_t tm,
                                        int stream, int wq, int lane, bool& ok) {
  using X = Shape<kMode, kD, kPair>;
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kMost = 3.402823466e38f;
  const int row = 32 * wq + lane;  // of the tile; also a key, where keys are prepared
  const int r = kPair ? 128 * stream + row : row;
  const uint32_t lanes = tm + ((uint32_t)(32 * wq) << 16);
  const uint32_t s_col = lanes + X::kColS + (uint32_t)stream * 128, o_col = lanes + X::kColO + (uint32_t)stream * 128;
  const float scale = p.scale * kLog2e;
  uint32_t mine = 0;  // tiles of this stream so far
  int base = 0;       // tiles of the CTA before the piece
  for (int rt = blockIdx.x % p.n_groups; rt < p.n_row_tiles; rt += p.n_groups) {
    TreeWalk walk;
    walk.start(p, sm.span);
    TreePiece w;
    while (walk.next(p, w)) {
      // ---- the queries; the scores of the last piece have all been read ----
      constexpr int kPerRow = kD / 8, kAll = X::kRows * kPerRow, kBatch = 4;
#pragma unroll 1
      for (int i0 = 128 * stream + row; i0 < kAll; i0 += 256 * kBatch) {
        uint4 v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + 256 * u, c = i % kPerRow;
          v[u] = make_uint4(0u, 0u, 0u, 0u);
          if (c * 8 < p.c.head_dim) {
            const TreeRow at = tree_row(p, w.hk, rt, i / kPerRow);
            if (at.exists)
              v[u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q.q) + w.b * p.q.q_seq_stride +
                                                     at.h * p.q.q_head_stride + at.t * p.q.q_row_stride + c * 8);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + 256 * u, rr = i / kPerRow, c = i % kPerRow;
          if constexpr (X::k8) {
            uint32_t h[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            uint32_t top = 0;  // largest exponent field of the row's kPerRow lanes
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max((h[e] >> 7) & 0xffu, (h[e] >> 23) & 0xffu));
#pragma unroll
            for (int off = kPerRow / 2; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
            const int up = top == 0 || top == 255 ? 0 : min(14 + 127 - (int)top, 120);
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = pack<true>(__uint_as_float(h[e] << 16) * f, __uint_as_float(h[e] & 0xffff0000u) * f);
            v[u] = make_uint4(h[0], h[1], h[2], h[3]);
            if (c == 0) sm.qf[rr] = __uint_as_float((uint32_t)(127 - up) << 23);
          }
          st_shared_v4(smem_u32(sm.q[rr >> 7]) + (uint32_t)((c >> 3) * 16384 + (rr & 127) * 128 + (((c & 7) ^ (rr & 7)) << 4)),
                       v[u].x, v[u].y, v[u].z, v[u].w);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&sm.bar_q);
      softmax_sync();  // qf
      const float unit = X::k8 ? scale * sm.qf[r] : scale;
      const TreeRow own = tree_row(p, w.hk, rt, r);
      float m = -INFINITY, l = 0.f;
      int v_exp = 0;  // exponent of the stream's V scales
      const bool busy = __any_sync(0xffffffffu, own.exists);  // else no row of the warp is anybody's
      const int count = w.k1 - w.k0;
      const int skip = kPair ? 0 : (stream - base % 2 + 2) % 2;
#pragma unroll 1
      for (int it = skip; it < count; it += kPair ? 1 : 2, ++mine) {
        const int j = base + it, ring = j % kRing;
        const bool first = it == skip;
        const int64_t i0 = (int64_t)(w.k0 + it) * kTreeKeys - w.s.ctx;  // of the tile's first key; >= 0: newest token
        // ---- the keys of the tile, one a thread ----
        wait_or_skip(ok, &sm.bar_side[ring], (uint32_t)(j / kRing) & 1);
        const uint4 vis = *reinterpret_cast<const uint4*>(sm.vis[ring]);
        const bool hidden = __any_sync(0xffffffffu, (vis.x & vis.y & vis.z & vis.w) != 0xffffffffu) || i0 + kTreeKeys > 0;
        bool prepared = false;
        if (X::k8 || p.c.bias || (guard && i0 + kTreeKeys > 0)) {  // the same in all warps of the stream: they meet at barriers
          prepared = true;
          float bias = p.c.bias ? sm.side[ring][0][row] : 0.f;
          if (bias > -INFINITY && bias < INFINITY) bias = fminf(fmaxf(bias * kLog2e, -kMost), kMost);
          const int64_t i = i0 + row;
          float v_nan = 1.f;  // NaN for such an e4m3 row: a factor of its V scale
          if (kMode != DCC_KV_INT8 && guard && i >= 0 && i < w.s.cnt) {
            // a newest value that is not finite: the rows that see it become NaN
            // (a row that was not finite when it was quantised has a NaN scale)
            const PageWalk pages{p.q.page_table + w.b * p.q.table_stride, p.c.n_pages, p.c.page_size, p.q.max_pages};
            int off = 0;
            const int64_t page = pages.page_of(i + w.s.ctx, off);
            if (page >= 0) {
              constexpr int kSize = X::k8 ? 1 : 2;
              const uint4* v = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(p.c.v) +
                                                              page_row(p.c, page, w.hk, off) * p.c.head_dim * kSize);
              for (int c = 0; c < p.c.head_dim * kSize / 16; ++c) {
                const uint4 x = __ldg(v + c);
                const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if constexpr (X::k8) {
                    if (((u[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) v_nan = __uint_as_float(0x7fc00000u);
                  } else {
                    if ((u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u) bias = __uint_as_float(0x7fc00000u);
                  }
                }
              }
            }
          }
          if constexpr (X::k8) {
            if (first) {
              float most = fmaxf(sm.side[ring][2][row], 0.f);
#pragma unroll
              for (int off = 16; off > 0; off /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
              if (lane == 0) sm.most[stream][wq] = most;
            }
          }
          group_sync(stream);  // the arrays of the last tile have been read
          sm.bias[stream][row] = bias;
          if constexpr (X::k8) {
            if (first) {
              v_exp = scale_exponent(fmaxf(fmaxf(sm.most[stream][0], sm.most[stream][1]), fmaxf(sm.most[stream][2], sm.most[stream][3])));
              if (row == 0) sm.up[stream] = v_exp;
            }
            const float own_vs = sm.side[ring][2][row] * two_to(kWeightUp - v_exp) * v_nan, vs = fmaxf(own_vs, kLeastScale);
            sm.ks[stream][row] = sm.side[ring][1][row];
            const bool huge = fabsf(bias) >= kHuge;
            sm.vs[stream][row] = own_vs < kLeastScale ? vs : huge && own_vs > kMostHuge ? kMostHuge : own_vs;
            sm.lift[stream][row] = huge ? bias : __log2f(vs) - kWeightUp + bias;
          }
          group_sync(stream);
        }
        wait_or_skip(ok, &sm.bar_s[stream], mine & 1);
        tc_fence_after();

        // keys 32 c .. 32 c + 31 that this row sees
        auto seen = [&](int c) {
          uint32_t see = c == 0 ? vis.x : c == 1 ? vis.y : c == 2 ? vis.z : vis.w;
          const int64_t i = i0 + 32 * c;
          if (i + 32 > 0) {
            const int from = i < 0 ? (int)-i : 0;  // the first newest token of the 32
            const int64_t some = w.s.cnt - i;
            const int to = some < 32 ? (int)(some < 0 ? 0 : some) : 32;
            uint32_t yes = from > 0 ? 0xffffffffu >> (32 - from) : 0u;
            if (own.exists)
              for (int x = from; x < to; ++x)
                if (tree_sees(p, w.b, own.t, i + x)) yes |= 1u << x;
            see &= yes;
          }
          return see;
        };
        float d[32];
        auto load = [&](int c) {
          tmem_ld32(s_col + 32 * c, reinterpret_cast<uint32_t*>(d));
          tmem_wait_ld();
        };
        // scores in powers of two with `add` of their keys (8-bit: always, else when
        // keys were prepared)
        auto scores = [&](int c, const float (&add)[128]) {
          load(c);
          if (X::k8 || prepared) {
#pragma unroll
            for (int x = 0; x < 32; x += 4) {
              const float4 b = *reinterpret_cast<const float4*>(&add[32 * c + x]);
              float4 k = make_float4(1.f, 1.f, 1.f, 1.f);
              if constexpr (X::k8) k = *reinterpret_cast<const float4*>(&sm.ks[stream][32 * c + x]);
              d[x] = fmaf(d[x] * unit, k.x, b.x);
              d[x + 1] = fmaf(d[x + 1] * unit, k.y, b.y);
              d[x + 2] = fmaf(d[x + 2] * unit, k.z, b.z);
              d[x + 3] = fmaf(d[x + 3] * unit, k.w, b.w);
            }
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) d[x] *= unit;
          }
        };
        // ---- largest score (with its V scale) ----
        if (busy) {
          float top = -INFINITY;
          const bool bare = !X::k8 && !prepared && !hidden && unit > 0.f;  // the scores themselves, scaled last
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (bare) {
              load(c);
#pragma unroll
              for (int x = 0; x < 32; ++x) mx[x & 3] = fmaxf(mx[x & 3], d[x]);
            } else {
              scores(c, X::k8 ? sm.lift[stream] : sm.bias[stream]);
              if (hidden) {
                const uint32_t see = seen(c);
#pragma unroll
                for (int x = 0; x < 32; ++x) d[x] = (see >> x) & 1 ? d[x] : -INFINITY;
              }
#pragma unroll
              for (int x = 0; x < 32; ++x) mx[x & 3] = fmaxf(mx[x & 3], d[x]);
            }
            top = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          }
          if (bare) top *= unit;
          const bool move = top > m + 8.f;
          if (__any_sync(0xffffffffu, move)) {
            const float f = move ? exp2f(m - top) : 1.f;  // 0 for the first score of a row
            if (!first) {
              wait_or_skip(ok, &sm.bar_o[stream], (mine - 1) & 1);
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < kD / 32; ++c) {
                tmem_ld32(o_col + 32 * c, reinterpret_cast<uint32_t*>(d));
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 32; ++x) d[x] *= f;
                tmem_st32(o_col + 32 * c, reinterpret_cast<const uint32_t*>(d));
              }
              tmem_wait_st();
            }
            l *= f;
            if (move) m = top;
          }
          // ---- weights, over the scores ----
          const float less = m == -INFINITY ? 0.f : m;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t see = 0xffffffffu;
            if (bare) {
              load(c);
#pragma unroll
              for (int x = 0; x < 32; ++x) d[x] = exp2_approx(fmaf(d[x], unit, -less));
            } else {
              if (X::k8 && !p.c.bias) {
                load(c);
#pragma unroll
                for (int x = 0; x < 32; x += 4) {
                  const float4 k = *reinterpret_cast<const float4*>(&sm.ks[stream][32 * c + x]);
                  d[x] = fmaf(d[x] * unit, k.x, -less);
                  d[x + 1] = fmaf(d[x + 1] * unit, k.y, -less);
                  d[x + 2] = fmaf(d[x + 2] * unit, k.z, -less);
                  d[x + 3] = fmaf(d[x + 3] * unit, k.w, -less);
                }
              } else {
                scores(c, sm.bias[stream]);
#pragma unroll
                for (int x = 0; x < 32; ++x) d[x] -= less;
              }
#pragma unroll
              for (int x = 0; x < 32; ++x) d[x] = exp2_approx(d[x]);
              if (hidden) {
                see = seen(c);
#pragma unroll
                for (int x = 0; x < 32; ++x) d[x] = (see >> x) & 1 ? d[x] : 0.f;
              }
            }
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < 32; ++x) sum[x & 3] += d[x];
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            uint32_t h[16];
            if constexpr (X::k8) {
#pragma unroll
              for (int x = 0; x < 32; x += 4) {
                float4 v = *reinterpret_cast<const float4*>(&sm.vs[stream][32 * c + x]);
                if (hidden) {  // a hidden key's scale may be NaN
                  v.x = (see >> x) & 1 ? v.x : 0.f;
                  v.y = (see >> (x + 1)) & 1 ? v.y : 0.f;
                  v.z = (see >> (x + 2)) & 1 ? v.z : 0.f;
                  v.w = (see >> (x + 3)) & 1 ? v.w : 0.f;
                }
                h[x / 2] = pack<true>(d[x] * v.x, d[x + 1] * v.y);
                h[x / 2 + 1] = pack<true>(d[x + 2] * v.z, d[x + 3] * v.w);
              }
            } else {
#pragma unroll
              for (int x = 0; x < 32; x += 2) h[x / 2] = pack<false>(d[x], d[x + 1]);
            }
            tmem_st16(s_col + 16 * c, h);  // over scores that have been read
          }
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(&sm.bar_p[stream]);
      }

      // ---- the piece is done ----
      if (skip < count) wait_or_skip(ok, &sm.bar_o[stream], (mine - 1) & 1);
      sm.ml[stream][row] = make_float2(m, l);
      softmax_sync();
      tc_fence_after();
      const bool other = !kPair && count > 1;  // both streams had a tile
      // of stream 0 and 1, or of this stream; `none`: the row saw no key there
      // (a factor of 0 is one: O may hold a NaN)
      float f0 = 1.f, f1 = 0.f, top = m, sum = l;
      bool none0 = l == 0.f, none1 = true;
      if constexpr (!kPair) {
        const float2 a = sm.ml[0][row], b = sm.ml[1][row];
        top = fmaxf(a.x, b.x);
        none0 = a.y == 0.f;
        none1 = b.y == 0.f;
        f0 = a.x == top ? 1.f : exp2f(a.x - top);
        f1 = b.x == top ? 1.f : exp2f(b.x - top);
        sum = (none0 ? 0.f : f0 * a.y) + (none1 ? 0.f : f1 * b.y);
      }
      float unit_o = 1.f;  // of O
      if constexpr (X::k8) {
        if (other) v_exp = max(sm.up[0], sm.up[1]);
        else if (!kPair) v_exp = sm.up[base % 2];
        unit_o = two_to(v_exp);
        if constexpr (kPair) {
          f0 *= two_to(-kWeightUp);
        } else {
          f0 *= two_to(max(sm.up[0] - v_exp - kWeightUp, -126));
          f1 *= two_to(max(sm.up[1] - v_exp - kWeightUp, -126));
        }
      }
      // a piece of one tile lies in one stream
      const uint32_t col_a = lanes + X::kColO + (uint32_t)(kPair ? stream : other ? 0 : base % 2) * 128;
      const bool second = !kPair && !other && base % 2;
      const float fa = second ? f1 : f0;
      const bool none_a = second ? none1 : none0;
      if (own.t >= w.s.cnt) sum = 0.f;  // a row that does not exist
      // -kMost: nothing but biases of the type's lowest value
      const float ln = top == -kMost ? -kMost : top * kLn2;
      const int64_t part = w.part >= 0 ? p.part_row(span, rt, w.part, r) : 0;
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      __nv_bfloat16* out = tree_out_row<__nv_bfloat16>(p, w.b, own);
      const bool wide = ((reinterpret_cast<uintptr_t>(out) & 15u) == 0);
      const int c_first = kPair ? 0 : stream * (kD / 64), c_last = kPair ? kD / 32 : (stream + 1) * (kD / 64);
#pragma unroll 1
      for (int c = c_first; c < c_last; ++c) {
        float d[32];
        tmem_ld32(col_a + 32 * c, reinterpret_cast<uint32_t*>(d));
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 32; ++x) d[x] = none_a ? 0.f : fa * d[x];
        if (other) {
          float e[32];
          tmem_ld32(col_a + 128 + 32 * c, reinterpret_cast<uint32_t*>(e));
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 32; ++x) d[x] = none1 ? d[x] : fmaf(f1, e[x], d[x]);
        }
        if (!own.exists) continue;
#pragma unroll
        for (int x = 0; x < 32; ++x) d[x] = d[x] * inv * unit_o;
        if (w.part >= 0) {
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            if (32 * c + x < p.c.head_dim)
              *reinterpret_cast<float4*>(p.part_o + part * kTreePartCols + 32 * c + x) = make_float4(d[x], d[x + 1], d[x + 2], d[x + 3]);
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) d[x] = sum != 0.f ? d[x] : 0.f;
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            if (32 * c + x >= p.c.head_dim) continue;
            const uint4 h = make_uint4(pack<false>(d[x], d[x + 1]), pack<false>(d[x + 2], d[x + 3]),
                                       pack<false>(d[x + 4], d[x + 5]), pack<false>(d[x + 6], d[x + 7]));
            if (wide) {
              *reinterpret_cast<uint4*>(out + 32 * c + x) = h;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) out[32 * c + x + e] = __float2bfloat16_rn(d[x + e]);
            }
          }
        }
      }
      if (own.exists && (kPair || stream == 0)) {
        if (w.part >= 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(ln, sum);
        else if (p.q.lse)
          p.q.lse[((int64_t)w.b * p.q.n_q_heads + own.h) * p.q.T + own.t] = sum != 0.f ? ln + logf(sum) : -INFINITY;
      }
      tc_fence_before();
      softmax_sync();  // ml, O and the queries are free again
      base += count;
    }
  }
}

template <int kMode, int kD, bool kPair>
__global__ void __launch_bounds__(Shape<kMode, kD, kPair>::kThreads, 1) tree_tc05_kernel(const __grid_constant__ TreeParams p,
                                                                                        const __grid_constant__ TreeMaps maps,
                                                                                        unsigned int* error,
                                                                                        unsigned int* report) {
  using X = Shape<kMode, kD, kPair>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  SmemOf<kMode, kD, kPair>& sm = *reinterpret_cast<SmemOf<kMode, kD, kPair>*>(smem_raw);
  if (smem_u32(smem_raw) & 1023u) {  // the swizzled tiles need it
    if (threadIdx.x == 0) record_give_up(error, report, 64u);
    return;
  }
  const int span = blockIdx.x / p.n_groups;
  tree_plan(p, span, sm.plan);
  if (threadIdx.x == 0) sm.span = sm.plan.plan;
  __syncthreads();
  const int rounds = (p.n_row_tiles - (int)(blockIdx.x % p.n_groups) + p.n_groups - 1) / p.n_groups;
  const int n = (int)(sm.span.end - sm.span.begin) * rounds;
  if (n == 0) return;  // the whole CTA
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform, also to the compiler
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < X::kSlots; ++i) {
      mbar_init(&sm.bar_full[i], X::k8 ? 4 : 1);
      mbar_init(&sm.bar_empty[i], 1);
      mbar_init(&sm.bar_raw[i], 1);
    }
    for (int i = 0; i < kRing; ++i) mbar_init(&sm.bar_side[i], X::k8 || p.c.bias ? 33 : 1);
    mbar_init(&sm.bar_q, 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.bar_s[i], 1);
      mbar_init(&sm.bar_p[i], 128);
      mbar_init(&sm.bar_o[i], 1);
    }
    mbar_init(&sm.bar_end, 1);
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sm.tmem;
  // rows may hide newest tokens from one another
  const bool guard = p.q.T > 1 || p.q.tree != nullptr;
  bool ok = true;
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(X::kRegsSoftmax));
    softmax<kMode, kD, kPair>(p, sm, guard, span, tm, warp >> 2, warp & 3, lane, ok);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(X::kRegsWork));
    if (warp == 8) issuer<kMode, kD, kPair>(p, sm, n, guard, tm, lane, ok);
    else if (warp <= 10) copies<kMode, kD, kPair>(p, maps, sm, warp == 10, n, lane, ok);
  } else if constexpr (X::k8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(X::kRegsWiden));
    widen_tiles<kMode, kD, kPair>(p, sm, warp >= 16, n, warp & 3, lane, ok);
  }
  if (!ok && lane == 0) record_give_up(error, report, 32u);
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tm, 512);
}

template <int kMode, int kD, bool kPair>
static int launch(const TreeParams& p, const TreeMaps& maps, unsigned int* error, cudaStream_t st) {
  using X = Shape<kMode, kD, kPair>;
  constexpr size_t smem = sizeof(SmemOf<kMode, kD, kPair>);
  static_assert(smem <= kSmemLimit, "shared memory");
  auto kernel = tree_tc05_kernel<kMode, kD, kPair>;
  DCC_CHECK(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "tree_tc05 smem"));
  // setmaxnreg draws on the launch's registers: fewer than planned would wait forever
  cudaFuncAttributes fa{};
  DCC_CHECK(check_cuda(cudaFuncGetAttributes(&fa, kernel), "tree_tc05 attributes"));
  if (fa.numRegs < X::kRegsLaunch)
    return fail(DCC_ERR_UNSUPPORTED, "tree_tc05: compiled with " + std::to_string(fa.numRegs) +
                                         " registers per thread, the register split needs " + std::to_string(X::kRegsLaunch));
  kernel<<<p.n_groups * p.n_spans, X::kThreads, smem, st>>>(p, maps, error, attn_error_report());
  return check_launch("tree_attention");
}
template <int kMode, int kD>
static int launch_rows(const TreeParams& p, const TreeMaps& maps, unsigned int* error, cudaStream_t st) {
  if constexpr (kMode != DCC_KV_BF16)
    if (p.n_rows == 256) return launch<kMode, kD, true>(p, maps, error, st);
  return launch<kMode, kD, false>(p, maps, error, st);
}
template <int kMode>
static int launch_d(const TreeParams& p, const TreeMaps& maps, unsigned int* error, cudaStream_t st) {
  return p.c.head_dim <= 64 ? launch_rows<kMode, 64>(p, maps, error, st) : launch_rows<kMode, 128>(p, maps, error, st);
}

}  // namespace tt

int launch_tree_tc05(const TreeParams& p, cudaStream_t st) {
  unsigned int* error = nullptr;
  DCC_CHECK(attn_error_flag_address(&error));
  tt::TreeMaps maps{};
  maps.page_rows = 8;
  while (maps.page_rows < 128 && p.c.page_size % (2 * maps.page_rows) == 0) maps.page_rows *= 2;
  switch (p.c.format) {
    case DCC_KV_INT8: return tt::launch_d<DCC_KV_INT8>(p, maps, error, st);
    case DCC_KV_E4M3: return tt::launch_d<DCC_KV_E4M3>(p, maps, error, st);
    default: break;
  }
  const uint64_t rows = (uint64_t)p.c.n_pages * p.c.n_kv_heads * p.c.page_size;
  DCC_CHECK(make_tmap_bf16_rows(&maps.k, p.c.k, p.c.head_dim, rows, maps.page_rows));
  DCC_CHECK(make_tmap_bf16_rows(&maps.v, p.c.v, p.c.head_dim, rows, maps.page_rows));
  return tt::launch_d<DCC_KV_BF16>(p, maps, error, st);
}

}  // namespace dcc
