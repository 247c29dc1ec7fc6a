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
//   warps 0-7    softmax, two warpgroups with half of the N rows each: thread =
//                key (TMEM lane), row sums per thread, added up at the end
//   warp  8      TMEM owner and MMA issuer
//   warp  9      queries of the next piece into shared memory
//   warp  10     page lookups and copies: the ring of K and V tiles stays full.
//                bf16 tiles come as TMA boxes of up to 128 rows of a page
//                straight into the layout of the MMA, 8-bit codes and scales as
//                bulk copies of rows that are neighbours in the page
//   warp  11     (bf16) clears the value rows of a tile that do not exist
//   warps 12-    (8-bit) 8 or 16 warps that widen codes, to bf16 for K and fp16
//                for V, both exactly.  A warp owns 16 or 8 rows of the tile and
//                reads their codes into registers from the place where it then
//                writes their values; the scales are applied to S and P in fp32
// Tile order in the ring: K0 K1 V0 K2 V1 ...; S^T is double buffered in TMEM,
// so the scores of tile j + 1 are ready while the softmax of tile j runs.
// The running max of a row is shared by all keys and moves (with O and the sums
// rescaled) only when a score passes it by 2^8.  P is rounded once for its MMA,
// to bf16 beside bf16 values (a relative 2^-9 of each weight) and to fp16 beside
// 8-bit ones (2^-12): there P carries the V scale, so the max is taken over
// score + log2(scale), which keeps P below 2^8 whatever the scales are.
//
// Bound: HBM for few rows (2 d bytes a key and head against 4 N d flops),
// tensor cores and softmax issue from ~100 rows on.
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
constexpr size_t kSmemLimit = 232448;

template <int kMode, int kD, int kN>  // cache format, padded head_dim, query rows
struct Shape {
  static constexpr bool k8 = kMode == DCC_KV_INT8 || kMode == DCC_KV_E4M3;
  static constexpr int kTile = 128 * kD * 2;          // bf16 K or V tile
  static constexpr int kBlocks = kD / 64;             // 64-column blocks of 128 swizzled rows
  static constexpr int kQ = kN * kD * 2;
  static constexpr int kP = kN <= 64 ? 16384 : 32768;
  static constexpr int kCols = kN / 2;                // rows of a softmax warpgroup
  static constexpr int kChunk = kCols < 32 ? kCols : 32;
  static constexpr int kChunks = kCols / kChunk;
  static constexpr uint32_t kColS = 0, kColO = 2 * kN;
  static constexpr int kTmem = kN == 16 ? 64 : kN == 32 ? 128 : kN == 64 ? 256 : 512;
  static constexpr int kArrays = k8 ? 3 : 1;          // bias; K and V scales
  static constexpr size_t kFixed = (size_t)kQ + kP + (size_t)kRing * kArrays * 512 + 5120;
  static constexpr int kFit = (int)((kSmemLimit - kFixed) / kTile);
  static constexpr int kSlots = kFit < 8 ? kFit : 8;
  static_assert(kSlots >= 4, "ring");
  // K tile j + kRing is loaded once the tile kSlots places before it in the
  // ring order has been consumed: that has to be V tile j or a later one, so
  // that the softmax of tile j no longer reads its scales
  static_assert(2 * kRing - 1 - kSlots >= 2, "scale ring");
  // widening is bound by the latency of its few instructions per code: 16
  // warps where the registers of the softmax allow it
  static constexpr int kWiden = !k8 ? 0 : kN <= 32 ? 16 : 8;
  static constexpr int kGroups = 3 + kWiden / 4;      // warpgroups
  static constexpr int kThreads = kGroups * 128;
  static constexpr int kRegsLaunch = 65536 / kThreads / 8 * 8;
  static constexpr int kRegsSoftmax = !k8 ? 192 : kN <= 32 ? 88 : kN == 64 ? 112 : 144;
  static constexpr int kRegsWork = !k8 ? 120 : kN <= 32 ? 72 : 80;  // issuer, queries, copies
  static constexpr int kRegsWiden = kN <= 32 ? 64 : kN == 64 ? 88 : 56;
  static_assert(2 * kRegsSoftmax + kRegsWork + (kGroups - 3) * kRegsWiden <= kGroups * kRegsLaunch, "register split");
};

template <typename X>
struct Smem {
  unsigned char slot[X::kSlots][X::kTile];
  unsigned char q[X::kQ];
  unsigned char p[X::kP];
  __align__(16) float side[kRing][X::kArrays][128];  // bias, k_scale, v_scale
  __align__(16) uint8_t vis[kRing][16];               // bits: keys that exist
  __align__(16) float m[2][64], corr[2][64];
  __align__(16) float red[2][4][64];
  uint64_t bar_raw[X::kSlots], bar_full[X::kSlots], bar_empty[X::kSlots], bar_side[kRing], bar_q, bar_qfree, bar_s[2], bar_p, bar_o, bar_end;
  uint32_t tmem;
  TreePlanSmem plan;
};

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
  if constexpr (N == 8) tmem_ld8(a, r);
  else if constexpr (N == 16) tmem_ld16(a, r);
  else tmem_ld32(a, r);
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t a, const uint32_t* r) {
  if constexpr (N == 8) tmem_st8(a, r);
  else if constexpr (N == 16) tmem_st16(a, r);
  else tmem_st32(a, r);
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
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Four 8-bit codes to four 16-bit floats (two per word), exactly: bf16 for K,
// fp16 for V.
template <int kMode, bool kHalf>
__device__ __forceinline__ uint2 widen(uint32_t w) {
  uint32_t o[2];
  if constexpr (kMode == DCC_KV_INT8 && kHalf) {
    const uint32_t u = w ^ 0x80808080u;  // code + 128
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t y = __byte_perm(u, 0x64646464u, i ? 0x4342 : 0x4140);  // 0x6400 | u = 1024 + u
      const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
      o[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
  } else if constexpr (kMode == DCC_KV_INT8) {
    // bits 0x4300 | b are 128 + b for b < 128; a code is b - 128 sign
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t y = __byte_perm(w, 0, i ? 0x4342 : 0x4140);  // code, 0, code, 0
      const uint32_t a = (y & 0x007f007fu) | 0x43004300u, b = (y & 0x00800080u) | 0x43004300u;
      const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
      o[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
  } else if constexpr (kHalf) {
    // exponent and mantissa in their fp16 places are the value times 2^-8
    // (bias 7 against 15), subnormals included: kValueUnit makes up for it
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t y = __byte_perm(w, 0, i ? 0x3424 : 0x1404);  // 0, code, 0, code
      o[i] = ((y & 0x7f007f00u) >> 1) | (y & 0x80008000u);
    }
  } else {
    // in their bf16 places the value times 2^-120 (bias 7 against 127)
    const uint32_t c = 0x7b807b80u;  // 2^120
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t y = __byte_perm(w, 0, i ? 0x3424 : 0x1404);
      const uint32_t a = ((y & 0x7f007f00u) >> 4) | (y & 0x80008000u);
      const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&c));
      o[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
  }
  return make_uint2(o[0], o[1]);
}
template <int kMode>
constexpr float kValueUnit = kMode == DCC_KV_E4M3 ? 256.f : 1.f;

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

// The ring order K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1).
struct Order {
  int k = 0, v = 0;
  __device__ __forceinline__ bool is_k(int n) const { return k < n && k <= v + 1; }
};

// ---- copies ----------------------------------------------------------------------------
template <int kMode, int kD, int kN>
__device__ __forceinline__ void copies(const TreeParams& p, const TreeMaps& maps, Smem<Shape<kMode, kD, kN>>& sm, int n, int lane,
                                       bool& ok) {
  using X = Shape<kMode, kD, kN>;
  const TreePlan& pl = sm.plan.plan;
  const uint32_t row_bytes = (uint32_t)p.c.head_dim * (X::k8 ? 1 : 2);
  const bool pow2 = (p.c.page_size & (p.c.page_size - 1)) == 0;
  const int shift = 31 - __clz(p.c.page_size);
  // rows of a copy: 8-bit rows shorter than their 128-byte place come in eights,
  // so that a warp's rows land within its own part of the tile
  const int rows = X::k8 && p.c.head_dim != 128 ? 8 : maps.page_rows;
  const int arrays = (X::k8 ? 2 : 0) + (p.c.bias ? 1 : 0);
  Tiles t;
  t.start(p, pl);
  // lane < 16: the page of rows 8 lane .. 8 lane + 7 of the next K tile, looked
  // up a tile ahead (a page holds all eight or none)
  int page = -1, off = 0, hk = 0, left = 0;
  auto fetch = [&]() {
    t.next(p, pl);
    const int pos = t.kt * kTreeKeys + 8 * lane;
    page = -1;
    left = (int)(t.w.s.total - pos);
    if (lane < 16 && left > 0) {
      const int s = pow2 ? pos >> shift : pos / p.c.page_size;
      off = pos - s * p.c.page_size;
      page = __ldg(p.q.page_table + (int64_t)t.w.b * p.q.table_stride + s);
    }
    hk = t.w.hk;
  };
  fetch();
  int row_a = -1, row_b = -1;  // cache rows of the latest K tile and the one before
  Order order;
  Place<X::kSlots> at;
#pragma unroll 1
  for (int i = 0; i < 2 * n; ++i) {
    const bool is_k = order.is_k(n);
    int row;
    if (is_k) {
      row_b = row_a;
      row_a = page >= 0 && page < p.c.n_pages ? (page * p.c.n_kv_heads + hk) * p.c.page_size + off : -1;
      row = row_a;
    } else {
      row = order.k == order.v + 2 ? row_b : row_a;
    }
    if (i >= X::kSlots) wait_or_skip(ok, &sm.bar_empty[at.slot], at.use ^ 1);
    // after a wait that ran out nothing new is set in flight (what was has
    // landed by then): the barriers are only passed on
    const bool real = ok && row >= 0;
    if (is_k) {
      const int ring = order.k % kRing;
      if (lane < 16) sm.vis[ring][lane] = row >= 0 ? (uint8_t)(left >= 8 ? 0xff : (1 << left) - 1) : (uint8_t)0;
      const bool lead = real && ((8 * lane) & (maps.page_rows - 1)) == 0;
      const uint32_t count = __popc(__ballot_sync(0xffffffffu, lead));
      if (lane == 0) mbar_expect_tx(&sm.bar_side[ring], count * (uint32_t)(maps.page_rows * 4 * arrays));
      __syncwarp();
      if (lead && arrays) {
        const uint32_t bytes = (uint32_t)maps.page_rows * 4;
        if (p.c.bias) bulk_load(smem_u32(&sm.side[ring][0][8 * lane]), p.c.bias + row, bytes, &sm.bar_side[ring]);
        if constexpr (X::k8) {
          bulk_load(smem_u32(&sm.side[ring][1][8 * lane]), p.c.k_scale + row, bytes, &sm.bar_side[ring]);
          bulk_load(smem_u32(&sm.side[ring][2][8 * lane]), p.c.v_scale + row, bytes, &sm.bar_side[ring]);
        }
      }
    }
    // bf16 keys need nothing further: a row that does not exist is hidden
    uint64_t* bar = !X::k8 && is_k ? &sm.bar_full[at.slot] : &sm.bar_raw[at.slot];
    const bool lead = real && ((8 * lane) & (rows - 1)) == 0;
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, lead));
    if (lane == 0) mbar_expect_tx(bar, count * (uint32_t)rows * (X::k8 ? row_bytes : X::kBlocks * 128));
    __syncwarp();
    if (lead) {
      const uint32_t dst = smem_u32(sm.slot[at.slot]) + (uint32_t)lane * 1024;
      if constexpr (X::k8) {
        bulk_load(dst, static_cast<const unsigned char*>(is_k ? p.c.k : p.c.v) + (int64_t)row * row_bytes,
                  (uint32_t)rows * row_bytes, bar);
      } else {
#pragma unroll
        for (int b = 0; b < X::kBlocks; ++b) tma_load_2d(dst + b * 16384, is_k ? &maps.k : &maps.v, bar, 64 * b, row);
      }
    }
    __syncwarp();
    if (is_k) {
      if (++order.k < n) fetch();
    } else {
      ++order.v;
    }
    at.next();
  }
}

// ---- bf16: value rows that must not meet a zero weight -----------------------------------
// Rows that do not exist hold whatever the page or the slot held, and newest
// values that are not finite must not reach rows that do not see them (0 * inf):
// both become zeros; the softmax marks the rows that do see the latter.
template <int kMode, int kD, int kN>
__device__ __forceinline__ void clear_values(const TreeParams& p, Smem<Shape<kMode, kD, kN>>& sm, int n, bool guard, int lane,
                                             bool& ok) {
  using X = Shape<kMode, kD, kN>;
  constexpr int kPerRow = kD / 8, kRowsPer = 32 / kPerRow;
  const int chunk = lane % kPerRow, sub = lane / kPerRow;
  Tiles t;
  t.start(p, sm.plan.plan);
  Order order;
  Place<X::kSlots> at;
  uint32_t use = 0;  // parity of bar_raw of each slot
#pragma unroll 1
  for (int i = 0; i < 2 * n; ++i) {
    if (order.is_k(n)) {
      ++order.k;
    } else {
      t.next(p, sm.plan.plan);
      const int64_t first = (int64_t)t.kt * kTreeKeys - t.w.s.ctx;  // of the tile, behind the context
      wait_or_skip(ok, &sm.bar_raw[at.slot], (use >> at.slot) & 1);
      use ^= 1u << at.slot;
      const uint4 vis = *reinterpret_cast<const uint4*>(sm.vis[order.v % kRing]);
      if ((vis.x & vis.y & vis.z & vis.w) != 0xffffffffu || (guard && first + kTreeKeys > 0)) {
        const uint32_t tile = smem_u32(sm.slot[at.slot]);
#pragma unroll 1
        for (int r = sub; r < kTreeKeys; r += kRowsPer) {
          const bool exists = (sm.vis[order.v % kRing][r >> 3] >> (r & 7)) & 1;
          if (exists && !(guard && first + r >= 0)) continue;
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
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.bar_full[at.slot]);
      ++order.v;
    }
    at.next();
  }
}

// ---- 8-bit: codes to values ----------------------------------------------------------------
template <int kMode, int kD, int kN>
__device__ __forceinline__ void widen_tiles(const TreeParams& p, Smem<Shape<kMode, kD, kN>>& sm, int n, int w, int lane, bool& ok) {
  using X = Shape<kMode, kD, kN>;
  constexpr int kPerRow = kD / 16;                  // 16-byte chunks of codes in a row
  constexpr int kRowsPer = 32 / kPerRow;            // rows of one step of the warp
  constexpr int kSteps = 128 / X::kWiden / kRowsPer;
  // lane -> (chunk, row of the step): eight lanes in a row write the eight
  // 16-byte banks of two rows, whose value chunks are two apart
  const int chunk = kPerRow == 8 ? (lane & 3) | ((lane >> 1) & 4) : lane & 3;
  const int sub = kPerRow == 8 ? ((lane >> 2) & 1) | ((lane >> 3) & 2) : lane >> 2;
  const bool chunk_real = chunk * 16 < p.c.head_dim;
  // offsets in a tile: codes, value chunks 2 chunk and 2 chunk + 1 (128-byte rows
  // of a 64-column block, chunks xor-ed with the row)
  uint32_t from[kSteps], to[kSteps][2];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int r = w * (128 / X::kWiden) + i * kRowsPer + sub;
    from[i] = (uint32_t)((r >> 3) * 1024 + (r & 7) * p.c.head_dim + chunk * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 2 * chunk + h;
      to[i][h] = (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    }
  }
  Order order;
  Place<X::kSlots> at;
#pragma unroll 1
  for (int i = 0; i < 2 * n; ++i) {
    const bool is_k = order.is_k(n);
    wait_or_skip(ok, &sm.bar_raw[at.slot], at.use);
    const uint32_t tile = smem_u32(sm.slot[at.slot]);
    uint4 raw[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) raw[s] = chunk_real ? ld_shared_v4(tile + from[s]) : make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();  // this warp alone reads and writes these rows
    auto store = [&](auto half) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t u[4] = {raw[s].x, raw[s].y, raw[s].z, raw[s].w};
        uint2 v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = widen<kMode, decltype(half)::value>(u[c]);
        st_shared_v4(tile + to[s][0], v[0].x, v[0].y, v[1].x, v[1].y);
        st_shared_v4(tile + to[s][1], v[2].x, v[2].y, v[3].x, v[3].y);
      }
    };
    if (is_k) store(std::false_type{});
    else store(std::true_type{});
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.bar_full[at.slot]);
    if (is_k) ++order.k;
    else ++order.v;
    at.next();
  }
}

// ---- MMA issuer ----------------------------------------------------------------------
template <int kMode, int kD, int kN>
__device__ __forceinline__ void issuer(const TreeParams& p, Smem<Shape<kMode, kD, kN>>& sm, int n, uint32_t tm, int lane,
                                       bool& ok) {
  using X = Shape<kMode, kD, kN>;
  const uint32_t id_s = idesc_bf16_f32(128, kN, 0, 0);
  const uint32_t id_o = X::k8 ? idesc_f16_f32(128, kN, 1, 1) : idesc_bf16_f32(128, kN, 1, 1);
  Tiles t;
  t.start(p, sm.plan.plan);
  Place<X::kSlots> at;
  uint32_t firsts = 0;  // bit j & 31: tile j opens a piece
  uint32_t pieces = 0;
  auto scores = [&](int j) {
    t.next(p, sm.plan.plan);
    firsts = (firsts & ~(1u << (j & 31))) | ((uint32_t)t.first << (j & 31));
    wait_or_skip(ok, &sm.bar_full[at.slot], at.use);
    if (t.first) {
      wait_or_skip(ok, &sm.bar_q, pieces & 1);
      ++pieces;
    }
    tc_fence_after();
    if (lane == 0) {
      const uint32_t k = smem_u32(sm.slot[at.slot]), q = smem_u32(sm.q);
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk)
        umma_ss(tm + X::kColS + (uint32_t)(j & 1) * kN, sdesc_sw128(k + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024),
                sdesc_sw128(q + (kk >> 2) * (kN * 128) + (kk & 3) * 32, 16, 1024), id_s, kk > 0);
      umma_commit(&sm.bar_s[j & 1]);
      umma_commit(&sm.bar_empty[at.slot]);
      if (t.last) umma_commit(&sm.bar_qfree);
    }
    __syncwarp();
    at.next();
  };
  scores(0);
  if (n > 1) scores(1);
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    wait_or_skip(ok, &sm.bar_full[at.slot], at.use);
    wait_or_skip(ok, &sm.bar_p, (uint32_t)(j & 1));
    tc_fence_after();
    if (lane == 0) {
      const uint32_t v = smem_u32(sm.slot[at.slot]), pr = smem_u32(sm.p);
      const bool first = (firsts >> (j & 31)) & 1;
      // with 64 columns both halves of the 128 MMA rows read the same block
      constexpr uint32_t kNextBlock = X::kBlocks == 2 ? 16384 : 0;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        umma_ss(tm + X::kColO, sdesc_sw128(v + kk * 2048, kNextBlock, 1024), sdesc_sw128(pr + kk * 2048, 16384, 1024), id_o,
                (first && kk == 0) ? 0u : 1u);
      umma_commit(&sm.bar_empty[at.slot]);
      umma_commit(&sm.bar_o);
    }
    __syncwarp();
    at.next();
    if (j + 2 < n) scores(j + 2);
  }
  // every MMA has finished before TMEM is freed, also after a wait that ran out
  if (lane == 0) umma_commit(&sm.bar_end);
  __syncwarp();
  if (!wait_all_lanes(&sm.bar_end, 0)) ok = false;
}

// ---- queries -------------------------------------------------------------------------
template <int kMode, int kD, int kN>
__device__ __forceinline__ void queries(const TreeParams& p, Smem<Shape<kMode, kD, kN>>& sm, int tid, bool& ok) {
  using X = Shape<kMode, kD, kN>;
  constexpr int kPerRow = kD / 8, kAll = kN * kPerRow, kThr = 32, kBatch = 8;
  const TreePlan& pl = sm.plan.plan;
  uint32_t piece = 0;
  for (int rt = blockIdx.x % p.n_groups; rt < p.n_row_tiles; rt += p.n_groups) {
    TreeWalk walk;
    walk.start(p, pl);
    TreePiece w;
    while (walk.next(p, w)) {
      bool free = piece == 0;
#pragma unroll 1
      for (int i0 = 0; i0 < kAll; i0 += kThr * kBatch) {
        uint4 v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * kThr + tid;
          const int r = i / kPerRow, c = i % kPerRow;
          v[u] = make_uint4(0u, 0u, 0u, 0u);
          if (i < kAll && c * 8 < p.c.head_dim) {
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
          const int i = i0 + u * kThr + tid;
          const int r = i / kPerRow, c = i % kPerRow;
          if (i < kAll)
            st_shared_v4(smem_u32(sm.q) + (c >> 3) * (kN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), v[u].x, v[u].y,
                         v[u].z, v[u].w);
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
__device__ __forceinline__ void softmax(const TreeParams& p, Smem<Shape<kMode, kD, kN>>& sm, int n, bool guard, int span,
                                        uint32_t tm, int wg, int wq, int lane, bool& ok) {
  using X = Shape<kMode, kD, kN>;
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kMost = 3.402823466e38f;
  const int key = 32 * wq + lane;  // of a tile; also the head column of O^T
  const int tid = key;
  const uint32_t lane_off = (uint32_t)(32 * wq) << 16;
  const int col0 = wg * X::kCols;
  const float scale = p.scale * kLog2e;
  const uint32_t p_row = smem_u32(sm.p) + (uint32_t)((key >> 3) * 1024 + (key & 7) * 128) + (uint32_t)(kN == 128 ? wg * 16384 : 0);
  const int p_chunk0 = kN == 128 ? 0 : col0 / 8;
  float l[X::kCols];
  Tiles t;
  t.start(p, sm.plan.plan);
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    t.next(p, sm.plan.plan);
    const uint32_t s_col = tm + lane_off + X::kColS + (uint32_t)(j & 1) * kN + col0;
    const uint32_t o_col = tm + lane_off + X::kColO + col0;
    if (t.first) {
#pragma unroll
      for (int c = 0; c < X::kCols; ++c) l[c] = 0.f;
      if (tid < X::kCols) sm.m[wg][tid] = -INFINITY;
      group_sync(wg);
    }
    // which rows see this thread's key
    const int ring = j % kRing;
    const int64_t i = (int64_t)t.kt * kTreeKeys + key - t.w.s.ctx;  // >= 0: newest token i
    bool broken = false;
    if (!X::k8 && guard && i >= 0 && i < t.w.s.cnt) {
      // is the value finite?  (8-bit rows that are not have a NaN scale)
      const PageWalk pages{p.q.page_table + t.w.b * p.q.table_stride, p.c.n_pages, p.c.page_size, p.q.max_pages};
      int off = 0;
      const int64_t page = pages.page_of(i + t.w.s.ctx, off);
      if (page >= 0) {
        const uint4* v = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.c.v) +
                                                        page_row(p.c, page, t.w.hk, off) * p.c.head_dim);
        for (int c = 0; c < p.c.head_dim / 8; ++c) {
          const uint4 x = __ldg(v + c);
          const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            broken = broken || (u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u;
        }
      }
    }
    uint64_t see = ~0ull;
    if (i >= 0) {
      see = 0;
      if (i < t.w.s.cnt) {
        int64_t row = (int64_t)t.rt * kN + col0;
        int64_t tok = row / p.group;
        int g = (int)(row - tok * p.group);
#pragma unroll 1
        for (int c = 0; c < X::kCols; ++c) {
          if (tok < p.q.T && tree_sees(p, t.w.b, tok, i)) see |= 1ull << c;
          if (++g == p.group) {
            g = 0;
            ++tok;
          }
        }
      }
    }
    wait_or_skip(ok, &sm.bar_side[ring], (uint32_t)((j / kRing) & 1));
    const bool exists = (sm.vis[ring][key >> 3] >> (key & 7)) & 1;
    float bias = 0.f, ks = scale, vs = 1.f;
    if (p.c.bias) {
      bias = sm.side[ring][0][key];
      if (bias > -INFINITY && bias < INFINITY) bias = fminf(fmaxf(bias * kLog2e, -kMost), kMost);
    }
    if constexpr (X::k8) {
      ks *= sm.side[ring][1][key];
      vs = sm.side[ring][2][key];
    }
    // the score at which the max moves, and what the V scale adds to it (from
    // 2^-100: rows that were never written have scale 0)
    const float lift = X::k8 ? log2f(fmaxf(vs, 7.888609e-31f)) : 0.f, most = 8.f - lift;
    if (!exists || bias == -INFINITY) see = 0;
    if (broken) bias = __uint_as_float(0x7fc00000u);  // the rows that see it become NaN
    const bool all = __all_sync(0xffffffffu, see == ~0ull) != 0;

    wait_or_skip(ok, &sm.bar_s[j & 1], (uint32_t)((j >> 1) & 1));
    tc_fence_after();
    float d[X::kChunk];
    // scores less the running max of chunk `ch`, 2^x units
    auto load = [&](int ch) {
      tmem_ld<X::kChunk>(s_col + ch * X::kChunk, reinterpret_cast<uint32_t*>(d));
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < X::kChunk; c += 4) {
        const float4 m = *reinterpret_cast<const float4*>(&sm.m[wg][ch * X::kChunk + c]);
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
    if (group_any(wg, over)) {
      // move the max of every row to the largest score so far, rescale
#pragma unroll 1
      for (int ch = 0; ch < X::kChunks; ++ch) {
        tmem_ld<X::kChunk>(s_col + ch * X::kChunk, reinterpret_cast<uint32_t*>(d));
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < X::kChunk; ++c) {
          const float x = fmaf(d[c], ks, bias) + lift;
          // floats as integers of the same order; NaN counts as nothing
          const int bits = __float_as_int((((see >> (ch * X::kChunk + c)) & 1) && x == x) ? x : -INFINITY);
          const int top = __reduce_max_sync(0xffffffffu, bits ^ ((bits >> 31) & 0x7fffffff));
          if (lane == 0) sm.red[wg][wq][ch * X::kChunk + c] = __int_as_float(top ^ ((top >> 31) & 0x7fffffff));
        }
      }
      group_sync(wg);
      if (tid < X::kCols) {
        const float m0 = sm.m[wg][tid];
        const float m1 = fmaxf(fmaxf(fmaxf(sm.red[wg][0][tid], sm.red[wg][1][tid]), fmaxf(sm.red[wg][2][tid], sm.red[wg][3][tid])), m0);
        sm.corr[wg][tid] = m0 == m1 ? 1.f : exp2f(m0 - m1);
        sm.m[wg][tid] = m1;
      }
      if (!t.first) wait_or_skip(ok, &sm.bar_o, (uint32_t)((j - 1) & 1));
      tc_fence_after();
      group_sync(wg);
#pragma unroll
      for (int ch = 0; ch < X::kChunks; ++ch) {
        if (!t.first) {
          tmem_ld<X::kChunk>(o_col + ch * X::kChunk, reinterpret_cast<uint32_t*>(d));
          tmem_wait_ld();
        }
#pragma unroll
        for (int c = 0; c < X::kChunk; ++c) {
          const float f = sm.corr[wg][ch * X::kChunk + c];
          l[ch * X::kChunk + c] *= f;
          d[c] *= f;
        }
        if (!t.first) tmem_st<X::kChunk>(o_col + ch * X::kChunk, reinterpret_cast<const uint32_t*>(d));
      }
      if (!t.first) tmem_wait_st();
      load(0);
    }
    // the products of the last tile have read P
    if (j > 0) wait_or_skip(ok, &sm.bar_o, (uint32_t)((j - 1) & 1));
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
    mbar_arrive(&sm.bar_p);
    if (!t.last) continue;

    // ---- the piece is done: sums over the keys, then O^T (thread = head column) ----
#pragma unroll
    for (int c = 0; c < X::kCols; ++c) {
      const float s = warp_sum(l[c]);
      if (lane == 0) sm.red[wg][wq][c] = s;
    }
    group_sync(wg);
    wait_or_skip(ok, &sm.bar_o, (uint32_t)(j & 1));
    tc_fence_after();
    const int64_t row0 = (int64_t)t.rt * kN + col0;
    int64_t tok = row0 / p.group;
    int g = (int)(row0 - tok * p.group);
    const int64_t part0 = t.w.part >= 0 ? p.part_row(span, t.rt, t.w.part, col0) : 0;
#pragma unroll 1
    for (int ch = 0; ch < X::kChunks; ++ch) {
      tmem_ld<X::kChunk>(o_col + ch * X::kChunk, reinterpret_cast<uint32_t*>(d));
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < X::kChunk; ++c) {
        const int col = ch * X::kChunk + c;
        float sum = (sm.red[wg][0][col] + sm.red[wg][1][col]) + (sm.red[wg][2][col] + sm.red[wg][3][col]);
        float m = sm.m[wg][col] * kLn2;
        if (sm.m[wg][col] == -kMost) m = -kMost;  // nothing but biases of the type's lowest value
        if (tok >= t.w.s.cnt) sum = 0.f;  // a row that does not exist
        if (tok < p.q.T) {
          if (t.w.part >= 0) {
            if (key < p.c.head_dim) p.part_o[(part0 + col) * kTreePartCols + key] = d[c] * kValueUnit<kMode>;
            if (key == 0) *reinterpret_cast<float2*>(p.part_ml + (part0 + col) * 2) = make_float2(m, sum);
          } else {
            const bool real = sum != 0.f;
            const TreeRow row{tok, t.w.hk * p.group + g, true};
            if (key < p.c.head_dim) tree_out_row<__nv_bfloat16>(p, t.w.b, row)[key] = __float2bfloat16_rn(real ? d[c] * kValueUnit<kMode> / sum : 0.f);
            if (key == 0 && p.q.lse)
              p.q.lse[((int64_t)t.w.b * p.q.n_q_heads + row.h) * p.q.T + tok] = real ? m + logf(sum) : -INFINITY;
          }
        }
        if (++g == p.group) {
          g = 0;
          ++tok;
        }
      }
    }
    group_sync(wg);  // red and m are free again
  }
}

template <int kMode, int kD, int kN>
__global__ void __launch_bounds__(Shape<kMode, kD, kN>::kThreads, 1) tree_tc05_kernel(const __grid_constant__ TreeParams p,
                                                                const __grid_constant__ TreeMaps maps, unsigned int* error) {
  using X = Shape<kMode, kD, kN>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem<X>& sm = *reinterpret_cast<Smem<X>*>(smem_raw);
  if (smem_u32(smem_raw) & 1023u) {  // the swizzled tiles need it
    if (threadIdx.x == 0) atomicOr(error, 64u);
    return;
  }
  const int span = blockIdx.x / p.n_groups;
  tree_plan(p, span, sm.plan);
  const int rounds = (p.n_row_tiles - (int)(blockIdx.x % p.n_groups) + p.n_groups - 1) / p.n_groups;
  const int n = (int)(sm.plan.plan.end - sm.plan.plan.begin) * rounds;
  if (n == 0) return;  // the whole CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < X::kSlots; ++i) {
      mbar_init(&sm.bar_full[i], X::k8 ? X::kWiden : 1);
      mbar_init(&sm.bar_empty[i], 1);
      mbar_init(&sm.bar_raw[i], 1);
    }
    for (int i = 0; i < kRing; ++i) mbar_init(&sm.bar_side[i], 1);
    mbar_init(&sm.bar_q, 32);
    mbar_init(&sm.bar_qfree, 1);
    mbar_init(&sm.bar_s[0], 1);
    mbar_init(&sm.bar_s[1], 1);
    mbar_init(&sm.bar_p, 256);
    mbar_init(&sm.bar_o, 1);
    mbar_init(&sm.bar_end, 1);
    fence_mbar_init();
  }
  if (warp == 8) {
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
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(X::kRegsSoftmax));
    softmax<kMode, kD, kN>(p, sm, n, guard, span, tm, warp >> 2, warp & 3, lane, ok);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(X::kRegsWork));
    if (warp == 8) issuer<kMode, kD, kN>(p, sm, n, tm, lane, ok);
    else if (warp == 9) queries<kMode, kD, kN>(p, sm, lane, ok);
    else if (warp == 10) copies<kMode, kD, kN>(p, maps, sm, n, lane, ok);
    else if (!X::k8) clear_values<kMode, kD, kN>(p, sm, n, guard, lane, ok);
  } else if constexpr (X::k8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(X::kRegsWiden));
    widen_tiles<kMode, kD, kN>(p, sm, n, warp - 12, lane, ok);
  }
  if (!ok && lane == 0) atomicOr(error, 32u);
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tm, X::kTmem);
}

template <int kMode, int kD, int kN>
static int launch(const TreeParams& p, const TreeMaps& maps, unsigned int* error, cudaStream_t st) {
  using X = Shape<kMode, kD, kN>;
  constexpr size_t smem = sizeof(Smem<X>);
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
    case 64: return launch<kMode, kD, 64>(p, maps, error, st);
    default: return launch<kMode, kD, 128>(p, maps, error, st);
  }
}
template <int kMode>
static int launch_d(const TreeParams& p, const TreeMaps& maps, unsigned int* error, cudaStream_t st) {
  return p.c.head_dim <= 64 ? launch_n<kMode, 64>(p, maps, error, st) : launch_n<kMode, 128>(p, maps, error, st);
}

}  // namespace tt

bool tree_tc05_supported(const dcc_kv_pages& c, const dcc_tree_query& q, int dtype) {
  // rows of 16-byte chunks, eight rows that never leave their page
  if (dtype != DCC_BF16 || c.format == DCC_KV_F32 || c.head_dim % 16 != 0 || c.page_size % 8 != 0) return false;
  auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
  for (const void* x : {(const void*)c.k, (const void*)c.v, (const void*)c.k_scale, (const void*)c.v_scale,
                        (const void*)c.bias, (const void*)q.q})
    if (!aligned(x)) return false;
  if (q.q_seq_stride % 8 || q.q_head_stride % 8 || q.q_row_stride % 8) return false;
  // positions, cache rows and the tiles of a CTA are counted in 32 bits
  const int64_t cap = (int64_t)q.max_pages * c.page_size;
  return cap < 0x7fffff00LL && c.n_pages * c.n_kv_heads * c.page_size < 0x7fffff00LL &&
         (double)q.n_seqs * (double)q.T * q.n_q_heads * (double)(cap + 128) < 1e15;
}

// Query rows per tile = N of the MMAs: the smallest that takes all rows, since
// a span reads its keys once for each tile; beyond 128 rows per-thread state no
// longer fits.
int tree_tc05_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

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
