// Tree attention over the paged cache on the 5th-gen tensor cores (tcgen05 +
// TMEM): bf16 queries, bf16 / int8 / e4m3 cache, head_dim a multiple of 16.
//
// The contractions are transposed, so that the 128 rows of an MMA are keys (or
// head columns) and the few query rows are its N:
//   S^T [128 keys, N rows]  = K [128, d]      Q^T        (both K-major)
//   O^T [d, N rows]        += V^T [d, 128]    P^T        (both MN-major)
// One token of 4 query heads costs an N = 16 MMA instead of 128 padded rows.
// A CTA walks over its span of key tiles (tree_attention.cuh), one warp or
// group of warps per role:
//   softmax      2 or 4 warpgroups (streams); tile j belongs to stream j mod
//                kStreams, which has its own S, P, O, running max and sums, so
//                the chain scores -> softmax -> values of one tile (about 2500
//                cycles, most of it waiting) runs beside those of the next;
//                the streams are added up at the end of a piece.  Thread = key
//                (TMEM lane), then head column
//   1 warp       S issuer and TMEM owner
//   1 warp       O issuer; for bf16 it clears value rows that do not exist
//   1 warp       queries of the next piece into shared memory
//   1 warp       page lookups and copies: the ring of K and V tiles stays full.
//                bf16 tiles come as TMA boxes of up to 128 rows of a page
//                straight into the layout of the MMA, 8-bit codes and scales as
//                bulk copies of rows that are neighbours in the page
//   8 warps      (8-bit) widen codes to fp16, exactly, one group K, the
//                other V.  A warp reads the codes of its 32 rows of the tile into
//                registers from the place where it then writes their values;
//                the scales are applied to S and P in fp32.  The queries are
//                held in fp16 too, each row scaled by a power of two that takes
//                its largest element to 2^14: bf16 digits fit, and what falls
//                below fp16's range is under 2^-39 of that element
// K and V tiles have rings of their own, so that every role sees every use of
// the barriers that it waits on; copies of K run two tiles ahead of V, so that
// a V tile does not sit in its ring while its softmax runs.
// The running max of a row moves (with O and the sums rescaled) only when a
// score passes it by 2^8.  P is rounded once for its MMA, to bf16 beside bf16
// values (a relative 2^-9 of each weight) and to fp16 beside 8-bit ones (2^-12):
// there P carries the V scale, so the max is taken over score + log2(scale),
// which keeps P below 2^8 whatever the scales are.
//
// Bound: HBM for few rows (2 d bytes a key and head against 4 N d flops).
//
// Waits are bounded (2 s).  After one has run out a role sets the error word
// and walks through the rest of its loop without waiting, so named barriers
// still match and TMEM is freed; the outputs are then invalid.
#include <string>
#include <type_traits>

#include "tc05.cuh"
#include "tree_attention.cuh"

namespace dcc {

using namespace tc05;

int attn_error_flag_address(unsigned int** out);

namespace tt {

constexpr int kRing = 8;  // scales and masks of the last K tiles
constexpr int kFetch = 4;   // K tiles between a page lookup and its use
constexpr int kLead = 2;    // tiles that copies of K run ahead of V
constexpr int kPieces = 8;  // queries of a piece are written once the scores of the one before are issued, at
                            // most kStreams tiles ahead of the softmax: 5 pieces of one tile
constexpr size_t kSmemLimit = 232448;

template <int kMode, int kD, int kN>  // cache format, padded head_dim, query rows
struct Shape {
  static constexpr bool k8 = kMode == DCC_KV_INT8 || kMode == DCC_KV_E4M3;
  static constexpr int kStreams = kN == 16 ? 4 : 2;
  static constexpr int kTile = 128 * kD * 2;          // K or V tile of 16-bit values
  static constexpr int kBlocks = kD / 64;             // 64-column blocks of 128 swizzled rows
  static constexpr int kQ = kN * kD * 2;
  // P: 128-byte rows (keys) of 64 columns; the streams of 16 or 32 columns share them
  static constexpr int kP = kN == 64 ? 2 * 16384 : 16384;
  static constexpr int kPStep = kN == 64 ? 16384 : 2 * kN;  // from stream to stream
  static constexpr int kChunk = kN < 32 ? kN : 32;    // columns held in registers at once
  static constexpr int kChunks = kN / kChunk;
  static constexpr int kOut = kN / kStreams;          // columns of a stream in the results
  static constexpr uint32_t kColS = 0, kColO = kStreams * kN;
  static constexpr int kTmem = 2 * kStreams * kN;
  static constexpr int kArrays = k8 ? 3 : 1;          // bias; K and V scales
  static constexpr size_t kFixed = (size_t)kQ + kP + (size_t)kRing * kArrays * 512 + 896 + kN * 128;
  static constexpr int kFit = (int)((kSmemLimit - kFixed) / kTile);
  static constexpr int kSlotsV = (kFit + 1) / 2 < 4 ? (kFit + 1) / 2 : 4, kSlotsK = kFit / 2 < 4 ? kFit / 2 : 4;
  static constexpr int kSlots = kSlotsK + kSlotsV;
  static_assert(kSlotsK >= 2, "rings");
  // K tile j + kRing is copied after V tile j + kRing - kLead - 1, which waited
  // for V tile j + kRing - kLead - 1 - kSlotsV to be consumed: that has to be
  // tile j or a later one, so that nobody reads its scales any more.  And a
  // place of the ring of scales belongs to one stream
  static_assert(kRing - kLead - 1 - kSlotsV >= 0 && kRing % kStreams == 0, "ring of scales");
  static constexpr int kWiden = k8 ? 8 : 0;
  static constexpr int kGroups = kStreams + 1 + kWiden / 4;  // warpgroups
  static constexpr int kThreads = kGroups * 128;
  static constexpr int kRegsLaunch = 65536 / kThreads / 8 * 8;
  static constexpr int kRegsSoftmax = k8 ? (kN == 16 ? 80 : kN == 32 ? 128 : 152) : (kN == 16 ? 96 : 192);
  static constexpr int kRegsWork = k8 ? 72 : (kN == 16 ? 88 : 112);  // issuers, queries, copies
  static constexpr int kRegsWiden = kN == 16 ? 56 : kN == 32 ? 72 : 48;
  static_assert(kStreams * kRegsSoftmax + kRegsWork + kWiden / 4 * kRegsWiden <= kGroups * kRegsLaunch, "register split");
  static_assert(kRegsWork <= kRegsLaunch && kRegsWiden <= kRegsLaunch && kRegsSoftmax >= kRegsLaunch, "register split");
};

template <typename X, int kN>
struct Smem {
  unsigned char slot[X::kSlots][X::kTile];
  unsigned char q[X::kQ];
  unsigned char p[X::kP];
  __align__(16) float side[kRing][X::kArrays][128];  // bias, k_scale, v_scale
  __align__(16) uint8_t vis[kRing][16];               // bits: keys that exist
  int32_t pages[kFetch][16];                          // of every eighth key of the next K tiles
  __align__(16) float qf[kPieces][kN];                // what undoes the scaling of a query row, by piece
  __align__(16) float m[X::kStreams][kN];
  __align__(16) float sum[X::kStreams][kN];           // while a piece runs: the last rescale
  union {
    float red[X::kStreams][4][kN];
    TreePlanSmem plan;                                // only before the roles begin
  };
  TreePlan span;
  uint64_t bar_raw[X::kSlots], bar_full[X::kSlots], bar_empty[X::kSlots], bar_side[kRing], bar_q, bar_qfree,
      bar_s[X::kStreams], bar_p[X::kStreams], bar_o[X::kStreams], bar_end;
  uint32_t tmem;
};
template <int kMode, int kD, int kN>
using SmemOf = Smem<Shape<kMode, kD, kN>, kN>;

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
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t a, uint32_t* r) {
  if constexpr (N == 4) tmem_ld4(a, r);
  else if constexpr (N == 8) tmem_ld8(a, r);
  else if constexpr (N == 16) tmem_ld16(a, r);
  else tmem_ld32(a, r);
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t a, const uint32_t* r) {
  if constexpr (N == 8) tmem_st8(a, r);
  else if constexpr (N == 16) tmem_st16(a, r);
  else tmem_st32(a, r);
}
template <int kStreams>
__device__ __forceinline__ void all_streams_sync() {
  asm volatile("bar.sync 5, %0;\n" ::"n"(128 * kStreams) : "memory");
}
__device__ __forceinline__ void group_sync(int wg) { asm volatile("bar.sync %0, 128;\n" ::"r"(1 + wg) : "memory"); }
// true when any thread of the warpgroup says so
__device__ __forceinline__ bool group_any(int wg, bool x) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)x), "r"(1 + wg)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Four 8-bit codes to four fp16 (two per word), exactly.
template <int kMode>
__device__ __forceinline__ uint2 widen(uint32_t w) {
  if constexpr (kMode == DCC_KV_INT8) {
    const uint32_t u = w ^ 0x80808080u;  // code + 128
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t y = __byte_perm(u, 0x64646464u, i ? 0x4342 : 0x4140);  // 0x6400 | u = 1024 + u
      const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
      o[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
    return make_uint2(o[0], o[1]);
  } else {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    return make_uint2((uint32_t)lo.x | (uint32_t)lo.y << 16, (uint32_t)hi.x | (uint32_t)hi.y << 16);
  }
}

// A place of the ring and the parity of its current use.
template <int kSlots>
struct Place {
  int slot = 0;
  uint32_t use = 0;
  __device__ __forceinline__ void next() {
    if (++slot == kSlots) {
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
template <int kMode, int kD, int kN>
__device__ __forceinline__ void copies(const TreeParams& p, const TreeMaps& maps, SmemOf<kMode, kD, kN>& sm, int n, int lane,
                                       bool& ok) {
  using X = Shape<kMode, kD, kN>;
  const TreePlan& pl = sm.span;
  const uint32_t row_bytes = (uint32_t)p.c.head_dim * (X::k8 ? 1 : 2);
  const bool pow2 = (p.c.page_size & (p.c.page_size - 1)) == 0;
  const int shift = 31 - __clz(p.c.page_size);
  // rows of a copy: 8-bit rows shorter than their 128-byte place come in eights,
  // so that a warp's rows land within its own part of the tile
  const int rows = X::k8 && p.c.head_dim != 128 ? 8 : maps.page_rows;
  const bool lead_side = lane < 16 && ((8 * lane) & (maps.page_rows - 1)) == 0;
  const bool lead_tile = lane < 16 && ((8 * lane) & (rows - 1)) == 0;
  const uint32_t side_bytes = (uint32_t)maps.page_rows * 4;
  const uint32_t side_all = side_bytes * (uint32_t)((X::k8 ? 2 : 0) + (p.c.bias ? 1 : 0));
  const uint32_t tile_all = (uint32_t)rows * (X::k8 ? row_bytes : X::kBlocks * 128);
  const uint32_t slot0 = smem_u32(sm.slot[0]) + (uint32_t)lane * 1024;
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
        cp_async4(smem_u32(&sm.pages[fetched % kFetch][lane]), p.q.page_table + (int64_t)t.w.b * p.q.table_stride + s);
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
  const int page_step = p.c.n_kv_heads * p.c.page_size;
  static_assert(kLead == 2, "rows of the last K tiles");
  int row0 = -1, row1 = -1, row2 = -1;  // of the latest K tile and the two before
  int kj = 0, vj = 0;      // next tiles
  Place<X::kSlotsK> at_k;
  Place<X::kSlotsV> at_v;
#pragma unroll 1
  while (vj < n) {
    const bool is_k = kj < n && kj <= vj + kLead;
    // after a wait that ran out nothing new is set in flight (what was has
    // landed by then): the barriers are only passed on
    int row, slot;
    if (is_k) {
      slot = at_k.slot;
      if (kj >= X::kSlotsK) wait_or_skip(ok, &sm.bar_empty[slot], at_k.use ^ 1);
      const int ring = kj % kRing;
      asm volatile("cp.async.wait_group %0;\n" ::"n"(kFetch - 1) : "memory");  // this lane's own page number
      row = -1;
      if (left[0] > 0) {
        const int page = sm.pages[kj % kFetch][lane];
        if (page >= 0 && page < p.c.n_pages) row = page * page_step + add[0];
      }
      if (lane < 16) {
        sm.vis[ring][lane] = row >= 0 ? (uint8_t)(left[0] >= 8 ? 0xff : (1 << left[0]) - 1) : (uint8_t)0;
      }
      const bool lead = ok && row >= 0 && lead_side;
      const uint32_t count = __popc(__ballot_sync(0xffffffffu, lead));
      __syncwarp();  // vis before the arrival
      if (lane == 0) mbar_expect_tx(&sm.bar_side[ring], count * side_all);
      __syncwarp();
      if (lead) {
        const uint32_t dst = smem_u32(&sm.side[ring][0][8 * lane]);
        if (p.c.bias) bulk_load(dst, p.c.bias + row, side_bytes, &sm.bar_side[ring]);
        if constexpr (X::k8) {
          bulk_load(dst + 512, p.c.k_scale + row, side_bytes, &sm.bar_side[ring]);
          bulk_load(dst + 1024, p.c.v_scale + row, side_bytes, &sm.bar_side[ring]);
        }
      }
      row2 = row1;
      row1 = row0;
      row0 = row;
    } else {
      slot = X::kSlotsK + at_v.slot;
      if (vj >= X::kSlotsV) wait_or_skip(ok, &sm.bar_empty[slot], at_v.use ^ 1);
      const int back = kj - 1 - vj;
      row = back == 0 ? row0 : back == 1 ? row1 : row2;
    }
    uint64_t* bar = X::k8 ? &sm.bar_raw[slot] : &sm.bar_full[slot];
    const bool lead = ok && row >= 0 && lead_tile;
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, lead));
    if (lane == 0) mbar_expect_tx(bar, count * tile_all);
    __syncwarp();
    if (lead) {
      const uint32_t dst = slot0 + (uint32_t)slot * X::kTile;
      if constexpr (X::k8) {
        bulk_load(dst, static_cast<const unsigned char*>(is_k ? p.c.k : p.c.v) + (int64_t)row * row_bytes, tile_all, bar);
      } else {
        const CUtensorMap* map = is_k ? &maps.k : &maps.v;
#pragma unroll
        for (int b = 0; b < X::kBlocks; ++b) tma_load_2d(dst + b * 16384, map, bar, 64 * b, row);
      }
    }
    if (is_k) {
      shift_down();
      fetch();
      ++kj;
      at_k.next();
    } else {
      ++vj;
      at_v.next();
    }
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");
}

// ---- 8-bit: codes to values ----------------------------------------------------------------
// Warps w = 0 .. 3 of the group for K or for V.
template <int kMode, int kD, int kN, bool kIsV>
__device__ __forceinline__ void widen_tiles(const TreeParams& p, SmemOf<kMode, kD, kN>& sm, int n, int w, int lane, bool& ok) {
  using X = Shape<kMode, kD, kN>;
  constexpr int kPerRow = kD / 16;                  // 16-byte chunks of codes in a row
  constexpr int kRowsPer = 32 / kPerRow;            // rows of one step of the warp: 4 or 8
  constexpr int kPair = 8 / kRowsPer;               // steps until the pattern of rows repeats, 1024 bytes on
  // lane -> (chunk, row of the step): eight lanes in a row write the eight
  // 16-byte banks of two rows, whose value chunks are two apart
  const int chunk = kPerRow == 8 ? (lane & 3) | ((lane >> 1) & 4) : lane & 3;
  const int sub = kPerRow == 8 ? ((lane >> 2) & 1) | ((lane >> 3) & 2) : lane >> 2;
  const bool chunk_real = chunk * 16 < p.c.head_dim;
  // offsets in a tile: codes, value chunks 2 chunk and 2 chunk + 1 (128-byte rows
  // of a 64-column block, chunks xor-ed with the row)
  uint32_t from[kPair], to[kPair][2];
#pragma unroll
  for (int i = 0; i < kPair; ++i) {
    const int r = 32 * w + i * kRowsPer + sub;
    from[i] = (uint32_t)((r >> 3) * 1024 + (r & 7) * p.c.head_dim + chunk * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 2 * chunk + h;
      to[i][h] = (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    }
  }
  constexpr int kFirst = kIsV ? X::kSlotsK : 0;
  Place<kIsV ? X::kSlotsV : X::kSlotsK> at;
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const int slot = kFirst + at.slot;
    wait_or_skip(ok, &sm.bar_raw[slot], at.use);
    const uint32_t tile = smem_u32(sm.slot[slot]);
    // whatever the slot held in rows that do not exist may be a NaN in e4m3,
    // which a zero weight would not hide
    uint32_t real = 0xffffffffu;
    if (kMode == DCC_KV_E4M3 && kIsV) real = *reinterpret_cast<const uint32_t*>(&sm.vis[j % kRing][4 * w]) >> sub;
#pragma unroll
    for (int half = 0; half < 2; ++half) {  // 16 rows at a time
      uint4 raw[2 * kPair];
#pragma unroll
      for (int s = 0; s < 2 * kPair; ++s)
        raw[s] = chunk_real && (kMode != DCC_KV_E4M3 || !kIsV || ((real >> (8 * (s / kPair + 2 * half) + s % kPair * kRowsPer)) & 1))
                     ? ld_shared_v4(tile + from[s % kPair] + (s / kPair + 2 * half) * 1024)
                     : make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();  // this warp alone reads and writes these rows
#pragma unroll
      for (int s = 0; s < 2 * kPair; ++s) {
        const uint2 a = widen<kMode>(raw[s].x), b = widen<kMode>(raw[s].y), c = widen<kMode>(raw[s].z), d = widen<kMode>(raw[s].w);
        const uint32_t on = (s / kPair + 2 * half) * 1024;
        st_shared_v4(tile + to[s % kPair][0] + on, a.x, a.y, b.x, b.y);
        st_shared_v4(tile + to[s % kPair][1] + on, c.x, c.y, d.x, d.y);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.bar_full[slot]);
    at.next();
  }
}

// ---- S issuer -----------------------------------------------------------------------
template <int kMode, int kD, int kN>
__device__ __forceinline__ void score_issuer(const TreeParams& p, SmemOf<kMode, kD, kN>& sm, int n, uint32_t tm, int lane,
                                             bool& ok) {
  using X = Shape<kMode, kD, kN>;
  const uint32_t id = X::k8 ? idesc_f16_f32(128, kN, 0, 0) : idesc_bf16_f32(128, kN, 0, 0);
  Tiles t;
  t.start(p, sm.span);
  Place<X::kSlotsK> at;
  uint32_t pieces = 0;
  const uint64_t q = desc_at(smem_u32(sm.q), 16);
  const uint32_t k0 = smem_u32(sm.slot[0]);
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    t.next(p, sm.span);
    const int stream = j % X::kStreams;
    if (t.first) {
      wait_or_skip(ok, &sm.bar_q, pieces & 1);
      ++pieces;
    }
    // the softmax has read the scores of the stream's last tile
    if (j >= X::kStreams) wait_or_skip(ok, &sm.bar_p[stream], (uint32_t)(j / X::kStreams - 1) & 1);
    wait_or_skip(ok, &sm.bar_full[at.slot], at.use);
    tc_fence_after();
    if (lane == 0) {
      const uint64_t k = desc_at(k0 + (uint32_t)at.slot * X::kTile, 16);
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk)
        umma_ss(tm + X::kColS + (uint32_t)stream * kN, k + ((kk >> 2) * 16384 + (kk & 3) * 32) / 16,
                q + ((kk >> 2) * (kN * 128) + (kk & 3) * 32) / 16, id, kk > 0);
      umma_commit(&sm.bar_s[stream]);
      umma_commit(&sm.bar_empty[at.slot]);
      if (t.last) umma_commit(&sm.bar_qfree);
    }
    __syncwarp();
    at.next();
  }
  // every MMA has finished before TMEM is freed, also after a wait that ran out
  if (lane == 0) umma_commit(&sm.bar_end);
  __syncwarp();
  if (!wait_all_lanes(&sm.bar_end, 0)) ok = false;
}

// ---- O issuer -----------------------------------------------------------------------
// bf16 value rows that do not exist hold whatever the page or the slot held,
// and newest values that are not finite must not reach rows that do not see
// them (0 * inf): both become zeros here; the softmax marks the rows that do
// see the latter.  (8-bit codes are always finite.)
template <int kMode, int kD, int kN>
__device__ __forceinline__ void clear_values(SmemOf<kMode, kD, kN>& sm, uint32_t tile, int ring, bool newest, int64_t first,
                                             int lane) {
  constexpr int kPerRow = kD / 8, kRowsPer = 32 / kPerRow;
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
        if ((u[c] & 0x7f80u) == 0x7f80u) u[c] &= 0xffff0000u;
        if ((u[c] & 0x7f800000u) == 0x7f800000u) u[c] &= 0x0000ffffu;
      }
    }
    st_shared_v4(a, u[0], u[1], u[2], u[3]);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

template <int kMode, int kD, int kN>
__device__ __forceinline__ void value_issuer(const TreeParams& p, SmemOf<kMode, kD, kN>& sm, int n, bool guard, uint32_t tm,
                                             int lane, bool& ok) {
  using X = Shape<kMode, kD, kN>;
  const uint32_t id = X::k8 ? idesc_f16_f32(128, kN, 1, 1) : idesc_bf16_f32(128, kN, 1, 1);
  // with 64 columns both halves of the 128 MMA rows read the same block
  constexpr uint32_t kNextBlock = X::kBlocks == 2 ? 16384 : 0;
  Tiles t;
  t.start(p, sm.span);
  Place<X::kSlotsV> at;
  const uint32_t v0 = smem_u32(sm.slot[X::kSlotsK]), p0 = smem_u32(sm.p);
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    t.next(p, sm.span);
    const int stream = j % X::kStreams;
    wait_or_skip(ok, &sm.bar_full[X::kSlotsK + at.slot], at.use);
    const uint32_t tile = v0 + (uint32_t)at.slot * X::kTile;
    if constexpr (!X::k8) {
      const int ring = j % kRing;
      wait_or_skip(ok, &sm.bar_side[ring], (uint32_t)(j / kRing) & 1);
      const uint4 vis = *reinterpret_cast<const uint4*>(sm.vis[ring]);
      const int64_t first = (int64_t)t.kt * kTreeKeys - t.w.s.ctx;  // of the tile, behind the context
      const bool newest = guard && first + kTreeKeys > 0;
      if ((vis.x & vis.y & vis.z & vis.w) != 0xffffffffu || newest)
        clear_values<kMode, kD, kN>(sm, tile, ring, newest, first, lane);
    }
    wait_or_skip(ok, &sm.bar_p[stream], (uint32_t)(j / X::kStreams) & 1);
    tc_fence_after();
    if (lane == 0) {
      const uint64_t v = desc_at(tile, kNextBlock), pr = desc_at(p0 + (uint32_t)stream * X::kPStep, 0);
      const bool first = t.kt - t.w.k0 < X::kStreams;  // of the stream in this piece
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        umma_ss(tm + X::kColO + (uint32_t)stream * kN, v + kk * 128, pr + kk * 128, id, (first && kk == 0) ? 0u : 1u);
      umma_commit(&sm.bar_empty[X::kSlotsK + at.slot]);
      umma_commit(&sm.bar_o[stream]);
    }
    __syncwarp();
    at.next();
  }
  if (lane == 0) umma_commit(&sm.bar_end);
  __syncwarp();
  if (!wait_all_lanes(&sm.bar_end, 0)) ok = false;
}

// ---- queries -------------------------------------------------------------------------
template <int kMode, int kD, int kN>
__device__ __forceinline__ void queries(const TreeParams& p, SmemOf<kMode, kD, kN>& sm, int lane, bool& ok) {
  using X = Shape<kMode, kD, kN>;
  constexpr int kPerRow = kD / 8, kAll = kN * kPerRow, kBatch = 4;
  const TreePlan& pl = sm.span;
  uint32_t piece = 0;
  for (int rt = blockIdx.x % p.n_groups; rt < p.n_row_tiles; rt += p.n_groups) {
    TreeWalk walk;
    walk.start(p, pl);
    TreePiece w;
    while (walk.next(p, w)) {
      bool free = piece == 0;
#pragma unroll 1
      for (int i0 = 0; i0 < kAll; i0 += 32 * kBatch) {
        uint4 v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * 32 + lane;
          const int r = i / kPerRow, c = i % kPerRow;
          v[u] = make_uint4(0u, 0u, 0u, 0u);
          if (c * 8 < p.c.head_dim) {
            const TreeRow row = tree_row(p, w.hk, rt, r);
            if (row.exists)
              v[u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q.q) + w.b * p.q.q_seq_stride +
                                                     row.h * p.q.q_head_stride + row.t * p.q.q_row_stride + c * 8);
          }
        }
        if (!free) {
          wait_or_skip(ok, &sm.bar_qfree, (piece - 1) & 1);
          free = true;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * 32 + lane;
          const int r = i / kPerRow, c = i % kPerRow;
          if constexpr (X::k8) {
            uint32_t h[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            uint32_t top = 0;  // largest exponent field of the row's kPerRow lanes
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max((h[e] >> 7) & 0xffu, (h[e] >> 23) & 0xffu));
#pragma unroll
            for (int o = kPerRow / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int up = top == 0 || top == 255 ? 0 : min(14 + 127 - (int)top, 120);
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              h[e] = pack_half(__uint_as_float(h[e] << 16) * f, __uint_as_float(h[e] & 0xffff0000u) * f);
            v[u] = make_uint4(h[0], h[1], h[2], h[3]);
            if (c == 0) sm.qf[piece % kPieces][r] = __uint_as_float((uint32_t)(127 - up) << 23);
          }
          st_shared_v4(smem_u32(sm.q) + (c >> 3) * (kN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), v[u].x, v[u].y, v[u].z,
                       v[u].w);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&sm.bar_q);
      ++piece;
    }
  }
}

// ---- softmax and results --------------------------------------------------------------
template <int kMode, int kD, int kN>
__device__ __forceinline__ void softmax(const TreeParams& p, SmemOf<kMode, kD, kN>& sm, bool guard, int span, uint32_t tm,
                                        int stream, int wq, int lane, bool& ok) {
  using X = Shape<kMode, kD, kN>;
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kMost = 3.402823466e38f;
  const int key = 32 * wq + lane;  // of a tile; also the head column of O^T
  const uint32_t lanes = tm + ((uint32_t)(32 * wq) << 16);
  const uint32_t s_col = lanes + X::kColS + (uint32_t)stream * kN;
  const uint32_t o_col = lanes + X::kColO + (uint32_t)stream * kN;
  const float scale = p.scale * kLog2e;
  const uint32_t p_row = smem_u32(sm.p) + (uint32_t)((key >> 3) * 1024 + (key & 7) * 128) +
                         (uint32_t)(kN == 64 ? stream * X::kPStep : 0);
  const int p_chunk0 = kN == 64 ? 0 : stream * kN / 8;
  uint32_t mine = 0;   // tiles of this stream so far
  int base = 0;        // tiles of the CTA before the piece
  uint32_t piece = 0;
  for (int rt = blockIdx.x % p.n_groups; rt < p.n_row_tiles; rt += p.n_groups) {
    TreeWalk walk;
    walk.start(p, sm.span);
    TreePiece w;
    while (walk.next(p, w)) {
      float l[kN];
#pragma unroll
      for (int c = 0; c < kN; ++c) l[c] = 0.f;
      if (key < kN) sm.m[stream][key] = -INFINITY;
      group_sync(stream);
      const int count = w.k1 - w.k0;
      const int skip = (stream - base % X::kStreams + X::kStreams) % X::kStreams;
      const float* qf = sm.qf[piece % kPieces];
#pragma unroll 1
      for (int it = skip; it < count; it += X::kStreams, ++mine) {
        const int j = base + it, ring = j % kRing;
        const bool first = it < X::kStreams;
        // which rows see this thread's key
        const int64_t i = (int64_t)(w.k0 + it) * kTreeKeys + key - w.s.ctx;  // >= 0: newest token i
        bool broken = false;
        uint64_t see = ~0ull;
        if (i >= 0) {
          see = 0;
          if (i < w.s.cnt) {
            int64_t row = (int64_t)rt * kN;
            int64_t tok = row / p.group;
            int g = (int)(row - tok * p.group);
#pragma unroll 1
            for (int c = 0; c < kN; ++c) {
              if (tok < p.q.T && tree_sees(p, w.b, tok, i)) see |= 1ull << c;
              if (++g == p.group) {
                g = 0;
                ++tok;
              }
            }
            if (!X::k8 && guard) {
              // is the value finite?  (8-bit rows that are not have a NaN scale)
              const PageWalk pages{p.q.page_table + w.b * p.q.table_stride, p.c.n_pages, p.c.page_size, p.q.max_pages};
              int off = 0;
              const int64_t page = pages.page_of(i + w.s.ctx, off);
              if (page >= 0) {
                const uint4* v = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.c.v) +
                                                                page_row(p.c, page, w.hk, off) * p.c.head_dim);
                for (int c = 0; c < p.c.head_dim / 8; ++c) {
                  const uint4 x = __ldg(v + c);
                  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    broken = broken || (u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u;
                }
              }
            }
          }
        }
        wait_or_skip(ok, &sm.bar_side[ring], (uint32_t)(j / kRing) & 1);
        const bool exists = (sm.vis[ring][key >> 3] >> (key & 7)) & 1;
        float bias = 0.f, ks = scale, vs = 1.f;
        if (p.c.bias) {
          bias = sm.side[ring][0][key];
          if (bias > -INFINITY && bias < INFINITY) bias = fminf(fmaxf(bias * kLog2e, -kMost), kMost);
        }
        // what the V scale adds to the score (from 2^-100: rows that were never
        // written have scale 0), and the score at which the max moves
        float lift = 0.f;
        if constexpr (X::k8) {
          ks *= sm.side[ring][1][key];
          vs = sm.side[ring][2][key];
          lift = __log2f(fmaxf(vs, 7.888609e-31f));
        }
        const float most = 8.f - lift;
        if (!exists || bias == -INFINITY) see = 0;
        if (broken) bias = __uint_as_float(0x7fc00000u);  // the rows that see it become NaN
        const bool all = __all_sync(0xffffffffu, see == ~0ull) != 0;

        wait_or_skip(ok, &sm.bar_s[stream], mine & 1);
        tc_fence_after();
        float d[X::kChunk];
        auto raw = [&](int ch) {
          tmem_ld<X::kChunk>(s_col + ch * X::kChunk, reinterpret_cast<uint32_t*>(d));
          tmem_wait_ld();
          if constexpr (X::k8) {
#pragma unroll
            for (int c = 0; c < X::kChunk; c += 4) {
              const float4 f = *reinterpret_cast<const float4*>(qf + ch * X::kChunk + c);
              d[c] *= f.x;
              d[c + 1] *= f.y;
              d[c + 2] *= f.z;
              d[c + 3] *= f.w;
            }
          }
        };
        // scores less the running max, in powers of two
        auto load = [&](int ch) {
          raw(ch);
#pragma unroll
          for (int c = 0; c < X::kChunk; c += 4) {
            const float4 m = *reinterpret_cast<const float4*>(&sm.m[stream][ch * X::kChunk + c]);
            d[c] = fmaf(d[c], ks, bias) - m.x;
            d[c + 1] = fmaf(d[c + 1], ks, bias) - m.y;
            d[c + 2] = fmaf(d[c + 2], ks, bias) - m.z;
            d[c + 3] = fmaf(d[c + 3], ks, bias) - m.w;
          }
        };
        bool over = false;
#pragma unroll
        for (int ch = X::kChunks - 1; ch >= 0; --ch) {
          load(ch);
          if (all) {
#pragma unroll
            for (int c = 0; c < X::kChunk; ++c) over = over || d[c] > most;
          } else {
#pragma unroll
            for (int c = 0; c < X::kChunk; ++c) over = over || (d[c] > most && ((see >> (ch * X::kChunk + c)) & 1));
          }
        }
        // (the vote also keeps a warp from moving the max that another still reads)
        if (group_any(stream, over)) {
          // move the max of every row to the largest score so far, rescale
#pragma unroll
          for (int ch = 0; ch < X::kChunks; ++ch) {
            raw(ch);
#pragma unroll
            for (int c = 0; c < X::kChunk; ++c) {
              const float x = fmaf(d[c], ks, bias) + lift;
              // floats as integers of the same order; NaN counts as nothing
              const int bits = __float_as_int((((see >> (ch * X::kChunk + c)) & 1) && x == x) ? x : -INFINITY);
              const int top = __reduce_max_sync(0xffffffffu, bits ^ ((bits >> 31) & 0x7fffffff));
              if (lane == 0) sm.red[stream][wq][ch * X::kChunk + c] = __int_as_float(top ^ ((top >> 31) & 0x7fffffff));
            }
          }
          group_sync(stream);
          if (key < kN) {
            const float m0 = sm.m[stream][key];
            const float m1 = fmaxf(fmaxf(fmaxf(sm.red[stream][0][key], sm.red[stream][1][key]),
                                         fmaxf(sm.red[stream][2][key], sm.red[stream][3][key])), m0);
            sm.sum[stream][key] = m0 == m1 ? 1.f : exp2f(m0 - m1);
            sm.m[stream][key] = m1;
          }
          if (!first) wait_or_skip(ok, &sm.bar_o[stream], (mine - 1) & 1);
          tc_fence_after();
          group_sync(stream);
#pragma unroll
          for (int ch = 0; ch < X::kChunks; ++ch) {
            if (!first) {
              tmem_ld<X::kChunk>(o_col + ch * X::kChunk, reinterpret_cast<uint32_t*>(d));
              tmem_wait_ld();
            }
#pragma unroll
            for (int c = 0; c < X::kChunk; ++c) {
              const float f = sm.sum[stream][ch * X::kChunk + c];
              l[ch * X::kChunk + c] *= f;
              d[c] *= f;
            }
            if (!first) tmem_st<X::kChunk>(o_col + ch * X::kChunk, reinterpret_cast<const uint32_t*>(d));
          }
          if (!first) tmem_wait_st();
          load(0);
        }
        // the stream's last products have read P
        if (mine > 0) wait_or_skip(ok, &sm.bar_o[stream], (mine - 1) & 1);
#pragma unroll
        for (int ch = 0; ch < X::kChunks; ++ch) {
          if (ch > 0) load(ch);
#pragma unroll
          for (int c8 = 0; c8 < X::kChunk; c8 += 8) {
            uint32_t h[4];
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
              float e0 = exp2_approx(d[c8 + c]), e1 = exp2_approx(d[c8 + c + 1]);
              if (!all) {
                const uint32_t two = (uint32_t)(see >> (ch * X::kChunk + c8 + c));
                e0 = two & 1 ? e0 : 0.f;
                e1 = two & 2 ? e1 : 0.f;
              }
              l[ch * X::kChunk + c8 + c] += e0;
              l[ch * X::kChunk + c8 + c + 1] += e1;
              if (X::k8) {  // a hidden key's scale may be NaN
                e0 = all || e0 != 0.f ? e0 * vs : 0.f;
                e1 = all || e1 != 0.f ? e1 * vs : 0.f;
              }
              h[c / 2] = X::k8 ? pack_half(e0, e1) : pack2(e0, e1);
            }
            const int chunk = p_chunk0 + (ch * X::kChunk + c8) / 8;
            st_shared_v4(p_row + (uint32_t)((chunk ^ (key & 7)) << 4), h[0], h[1], h[2], h[3]);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&sm.bar_p[stream]);
      }

      // ---- the piece is done: sums over the keys, streams together ----
#pragma unroll
      for (int c = 0; c < kN; ++c) {
        const float s = warp_sum(l[c]);
        if (lane == 0) sm.red[stream][wq][c] = s;
      }
      group_sync(stream);
      if (key < kN)
        sm.sum[stream][key] = (sm.red[stream][0][key] + sm.red[stream][1][key]) + (sm.red[stream][2][key] + sm.red[stream][3][key]);
      if (skip < count) wait_or_skip(ok, &sm.bar_o[stream], (mine - 1) & 1);
      all_streams_sync<X::kStreams>();
      tc_fence_after();
      // O^T: thread = head column, this stream's share of the rows
      const int64_t row0 = (int64_t)rt * kN + stream * X::kOut;
      int64_t tok = row0 / p.group;
      int g = (int)(row0 - tok * p.group);
      const int64_t part0 = w.part >= 0 ? p.part_row(span, rt, w.part, stream * X::kOut) : 0;
      constexpr int kSub = X::kOut < 8 ? X::kOut : 8;
#pragma unroll 1
      for (int c0 = 0; c0 < X::kOut; c0 += kSub) {
        float o[kSub], total[kSub], top[kSub];
#pragma unroll
        for (int c = 0; c < kSub; ++c) {
          o[c] = total[c] = 0.f;
          top[c] = -INFINITY;
#pragma unroll
          for (int s = 0; s < X::kStreams; ++s) top[c] = fmaxf(top[c], sm.m[s][stream * X::kOut + c0 + c]);
        }
#pragma unroll
        for (int s = 0; s < X::kStreams; ++s) {
          if ((s - base % X::kStreams + X::kStreams) % X::kStreams >= count) continue;  // no tile of the piece
          float part[kSub];
          tmem_ld<kSub>(lanes + X::kColO + (uint32_t)(s * kN + stream * X::kOut + c0), reinterpret_cast<uint32_t*>(part));
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < kSub; ++c) {
            const int col = stream * X::kOut + c0 + c;
            const float ls = sm.sum[s][col];
            if (ls != 0.f) {  // that stream saw a key of this row
              const float f = sm.m[s][col] == top[c] ? 1.f : exp2f(sm.m[s][col] - top[c]);
              o[c] = fmaf(f, part[c], o[c]);
              total[c] = fmaf(f, ls, total[c]);
            }
          }
        }
#pragma unroll
        for (int c = 0; c < kSub; ++c) {
          const float sum = tok < w.s.cnt ? total[c] : 0.f;  // a row that does not exist has none
          // -kMost: nothing but biases of the type's lowest value
          const float m = top[c] == -kMost ? -kMost : top[c] * kLn2;
          if (tok < p.q.T) {
            if (w.part >= 0) {
              if (key < p.c.head_dim) p.part_o[(part0 + c0 + c) * kTreePartCols + key] = o[c];
              if (key == 0) *reinterpret_cast<float2*>(p.part_ml + (part0 + c0 + c) * 2) = make_float2(m, sum);
            } else {
              const TreeRow row{tok, w.hk * p.group + g, true};
              if (key < p.c.head_dim)
                tree_out_row<__nv_bfloat16>(p, w.b, row)[key] = __float2bfloat16_rn(sum != 0.f ? o[c] / sum : 0.f);
              if (key == 0 && p.q.lse)
                p.q.lse[((int64_t)w.b * p.q.n_q_heads + row.h) * p.q.T + tok] = sum != 0.f ? m + logf(sum) : -INFINITY;
            }
          }
          if (++g == p.group) {
            g = 0;
            ++tok;
          }
        }
      }
      tc_fence_before();
      all_streams_sync<X::kStreams>();  // m, sums and O are free again
      base += count;
      ++piece;
    }
  }
}

template <int kMode, int kD, int kN>
__global__ void __launch_bounds__(Shape<kMode, kD, kN>::kThreads, 1) tree_tc05_kernel(const __grid_constant__ TreeParams p,
                                                                                      const __grid_constant__ TreeMaps maps,
                                                                                      unsigned int* error) {
  using X = Shape<kMode, kD, kN>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  SmemOf<kMode, kD, kN>& sm = *reinterpret_cast<SmemOf<kMode, kD, kN>*>(smem_raw);
  if (smem_u32(smem_raw) & 1023u) {  // the swizzled tiles need it
    if (threadIdx.x == 0) atomicOr(error, 64u);
    return;
  }
  const int span = blockIdx.x / p.n_groups;
  tree_plan(p, span, sm.plan);
  if (threadIdx.x == 0) sm.span = sm.plan.plan;
  __syncthreads();
  const int rounds = (p.n_row_tiles - (int)(blockIdx.x % p.n_groups) + p.n_groups - 1) / p.n_groups;
  const int n = (int)(sm.span.end - sm.span.begin) * rounds;
  if (n == 0) return;  // the whole CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < X::kSlots; ++i) {
      mbar_init(&sm.bar_full[i], X::k8 ? 4 : 1);
      mbar_init(&sm.bar_empty[i], 1);
      mbar_init(&sm.bar_raw[i], 1);
    }
    for (int i = 0; i < kRing; ++i) mbar_init(&sm.bar_side[i], 1);
    mbar_init(&sm.bar_q, 32);
    mbar_init(&sm.bar_qfree, 1);
    for (int i = 0; i < X::kStreams; ++i) {
      mbar_init(&sm.bar_s[i], 1);
      mbar_init(&sm.bar_p[i], 128);
      mbar_init(&sm.bar_o[i], 1);
    }
    mbar_init(&sm.bar_end, 2);
    fence_mbar_init();
  }
  constexpr int kWork = 4 * X::kStreams;  // first warp behind the softmax
  if (warp == kWork) {
    tmem_alloc(&sm.tmem, X::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sm.tmem;
  // rows may hide newest tokens from one another
  const bool guard = p.q.T > 1 || p.q.tree != nullptr;
  bool ok = true;
  if (warp < kWork) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(X::kRegsSoftmax));
    softmax<kMode, kD, kN>(p, sm, guard, span, tm, warp >> 2, warp & 3, lane, ok);
  } else if (warp < kWork + 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(X::kRegsWork));
    if (warp == kWork) score_issuer<kMode, kD, kN>(p, sm, n, tm, lane, ok);
    else if (warp == kWork + 1) value_issuer<kMode, kD, kN>(p, sm, n, guard, tm, lane, ok);
    else if (warp == kWork + 2) queries<kMode, kD, kN>(p, sm, lane, ok);
    else copies<kMode, kD, kN>(p, maps, sm, n, lane, ok);
  } else if constexpr (X::k8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(X::kRegsWiden));
    if (warp < kWork + 8) widen_tiles<kMode, kD, kN, false>(p, sm, n, warp & 3, lane, ok);
    else widen_tiles<kMode, kD, kN, true>(p, sm, n, warp & 3, lane, ok);
  }
  if (!ok && lane == 0) atomicOr(error, 32u);
  tc_fence_before();
  __syncthreads();
  if (warp == kWork) tmem_dealloc(tm, X::kTmem);
}

template <int kMode, int kD, int kN>
static int launch(const TreeParams& p, const TreeMaps& maps, unsigned int* error, cudaStream_t st) {
  using X = Shape<kMode, kD, kN>;
  constexpr size_t smem = sizeof(SmemOf<kMode, kD, kN>);
  static_assert(smem <= kSmemLimit, "shared memory");
  auto kernel = tree_tc05_kernel<kMode, kD, kN>;
  DCC_CHECK(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "tree_tc05 smem"));
  // setmaxnreg draws on the launch's registers: fewer than planned would wait forever
  cudaFuncAttributes fa{};
  DCC_CHECK(check_cuda(cudaFuncGetAttributes(&fa, kernel), "tree_tc05 attributes"));
  if (fa.numRegs < X::kRegsLaunch)
    return fail(DCC_ERR_UNSUPPORTED, "tree_tc05: compiled with " + std::to_string(fa.numRegs) +
                                         " registers per thread, the register split needs " + std::to_string(X::kRegsLaunch));
  kernel<<<p.n_groups * p.n_spans, X::kThreads, smem, st>>>(p, maps, error);
  return check_launch("tree_attention");
}
template <int kMode, int kD>
static int launch_n(const TreeParams& p, const TreeMaps& maps, unsigned int* error, cudaStream_t st) {
  switch (p.n_rows) {
    case 16: return launch<kMode, kD, 16>(p, maps, error, st);
    case 32: return launch<kMode, kD, 32>(p, maps, error, st);
    default: return launch<kMode, kD, 64>(p, maps, error, st);
  }
}
template <int kMode>
static int launch_d(const TreeParams& p, const TreeMaps& maps, unsigned int* error, cudaStream_t st) {
  return p.c.head_dim <= 64 ? launch_n<kMode, 64>(p, maps, error, st) : launch_n<kMode, 128>(p, maps, error, st);
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
