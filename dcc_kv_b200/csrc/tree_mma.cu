// Tree attention over the paged cache for few query rows (up to 16 per KV
// head): bf16 queries, bf16 / int8 / e4m3 cache, head_dim a multiple of 16.
//
// With few rows every key is used for so little arithmetic that HBM is the
// bound, and what a kernel has to save is instructions per key.  Here every
// warp works alone on 16 keys at a time: it copies them (cp.async, 512 bytes in
// a row) into a ring of its own and widens codes in registers, on their way to
// the MMA -- no barriers between warps, no second trip through shared memory
// for widened codes.  The contractions are register MMAs
// (m16n8k16) with keys, then head columns, as the 16 rows and query rows as the
// 8 columns -- four query heads and one token fill half of a tile:
//   S^T [16 keys, 8 rows]  += K Q^T    the k index runs over d in the order in
//                                      which a lane's 16-byte chunks hold it
//   O^T [16 cols, 8 rows]  += V^T P^T  rows n and n + 8 of tile i stand for
//                                      elements 2 i and 2 i + 1 of the chunk of V
//                                      that lane group n holds, so pairs of keys
//                                      are joined by byte permutes
// (P^T is transposed between the two by movmatrix.)
// Codes become fp16, exactly; scales act on S and P in fp32.  Beside them the
// queries are held in fp16 too, each row scaled by a power of two that takes
// its largest element to 2^14: bf16 digits fit, and what falls below fp16's
// range is under 2^-39 of that element.
// Each warp keeps a running max that moves when a score passes it by 2^8, its
// sums and O in registers; the warps are added up at the end of a piece.  P is
// rounded once, to bf16 beside bf16 values (a relative 2^-8 of each weight), to
// fp16 beside codes (2^-11): there P carries the V scale, so the max is taken
// over score + log2(scale), in units that keep it below 2^14 (kWeightUp in
// tree_attention.cuh; below 2^-20 of the largest fp16 is subnormal and holds P
// to 2^-31 of that).
// Measured: 16 sequences of 8192 tokens, 4 query heads on each of 8 KV heads of
// 128: int8 73 us or 3.8 TB/s, e4m3 83 us, bf16 102 us or 5.3 TB/s; with 16 rows
// per KV head int8 108, bf16 113 us.  Beside 8-bit codes the bound is the latency
// of the widening's dependent chains with three warps a scheduler (the registers
// allow no more, and 16 warps were slower, 81 against 75 us): 550 to 600
// instructions a warp and 16 keys fill 51 to 56 % of the issue slots.  Lines of 512
// bytes a copy instead of one row a lane took a quarter off; heads of 96, which
// are copied row by row and padded to 128 columns, take 87 us (int8) and 86 (bf16)
// for three quarters of the bytes, heads of 64 take 60 (int8).
#include <string>
#include <type_traits>

#include "tree_attention.cuh"

namespace dcc {
namespace tm {

constexpr size_t kSmemLimit = 232448;

template <int kMode, int kD, int kNT>  // cache format, padded head_dim, 8-row tiles
struct Shape {
  static constexpr bool k8 = kMode != DCC_KV_BF16;
  // as many warps as the registers of a warp and the ring (64 KB and more in
  // flight) allow
  static constexpr int kWarps = k8 || kNT == 1 ? 12 : 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kE = k8 ? 16 : 8;             // elements of a 16-byte chunk
  static constexpr int kKC = kD / (4 * kE);          // K chunks of a lane and key
  static constexpr int kVC = k8 ? 1 : kD / 64;       // V chunks of a lane and key
  static constexpr int kVB = k8 ? kD / 8 : 16;       // bytes of one
  static constexpr int kSteps = kD / 16;             // k steps of S
  static constexpr int kTiles = kD / 16;             // 16-column tiles of O
  static constexpr int kRowBytes = kD * (k8 ? 1 : 2), kPerRow = kRowBytes / 16;  // 16-byte chunks of a row
  static constexpr int kK = 16 * kRowBytes, kV = kK, kSide = 3 * 64;
  static constexpr int kStage = kK + kV + kSide;     // 16 keys of a warp
  // operands of the queries: in registers, or, where O takes those, in shared memory
  static constexpr bool kQShared = k8 && kNT > 1;
  static constexpr int kQ = kQShared ? kNT * kSteps * 256 : 16;
  static constexpr int kSum = kWarps * 2 * kD * 4;   // O of two rows of every warp
  static constexpr size_t kFixed = kSum + (size_t)kWarps * 8 * kNT * 8 + kWarps * 68 + kQ + 1024;
  static constexpr int kFit = (int)((kSmemLimit - kFixed) / ((size_t)kStage * kWarps));
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static_assert(kStages >= 2, "ring");
};

template <typename X, int kNT>
struct Smem {
  unsigned char ring[X::kWarps][X::kStages][X::kStage];
  float sum[X::kSum / 4];
  __align__(16) unsigned char q[X::kQ];
  float m[X::kWarps][8 * kNT], l[X::kWarps][8 * kNT];
  int up[X::kWarps];  // exponent of the warp's V scales (see kWeightUp)
  int2 info[X::kWarps][X::kStages];  // keys that exist (16 bits), first key behind the context
  TreePlanSmem plan;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t a, uint32_t* w) {
  if constexpr (kWords == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
  else
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "r"(a) : "memory");
}
template <int kWords>
__device__ __forceinline__ void store_words(uint32_t a, const uint32_t* w) {
  if constexpr (kWords == 4)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(a), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
  else
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(a), "r"(w[0]), "r"(w[1]) : "memory");
}
template <bool kHalf>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (kHalf)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit numbers held two to a lane.
__device__ __forceinline__ uint32_t transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float load_one(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(a) : "memory");
  return v;
}
// Code `q` of a and of b as a pair of fp16.
template <int kMode>
__device__ __forceinline__ uint32_t join_codes(uint32_t a, uint32_t b, int q) {
  if constexpr (kMode == DCC_KV_INT8) {
    const uint32_t y = __byte_perm(a, b, 0x0400u + 0x0101u * q);  // a.q, ., b.q, .
    return less_1152((y & 0x00ff00ffu) ^ 0x64806480u);
  } else {
    return from_e4m3(__byte_perm(a, b, 0x0040u + 0x0011u * q) & 0xffffu);
  }
}

// The position of a warp's next chunk of 16 keys.
struct Cursor {
  TreeWalk walk;
  TreePiece w;
  int rt, pos, end;  // end of the piece
  __device__ __forceinline__ void open(const TreeParams& p, const TreePlan& pl) {
    if (!walk.next(p, w)) {
      rt += p.n_groups;
      walk.start(p, pl);
      walk.next(p, w);
    }
    pos = w.k0 * kTreeKeys;
    end = w.k1 * kTreeKeys;
  }
  __device__ __forceinline__ void start(const TreeParams& p, const TreePlan& pl) {
    rt = blockIdx.x % p.n_groups;
    walk.start(p, pl);
    open(p, pl);
  }
  // over `keys` more of the CTA's line, which does not end before them
  __device__ __forceinline__ void move(const TreeParams& p, const TreePlan& pl, int keys) {
    pos += keys;
    while (pos >= end) {
      const int over = pos - end;
      open(p, pl);
      pos += over;
    }
  }
};

template <int kMode, int kD, int kNT>
__global__ void __launch_bounds__(Shape<kMode, kD, kNT>::kThreads, 1) tree_mma_kernel(const __grid_constant__ TreeParams p) {
  using X = Shape<kMode, kD, kNT>;
  constexpr bool k8 = X::k8;
  constexpr int kRows = 8 * kNT, S = X::kStages, NW = X::kWarps;
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kMost = 3.402823466e38f;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Smem<X, kNT>& sm = *reinterpret_cast<Smem<X, kNT>*>(smem_raw);
  const int span = blockIdx.x / p.n_groups;
  tree_plan(p, span, sm.plan);
  const TreePlan pl = sm.plan.plan;
  const int rounds = (p.n_row_tiles - (int)(blockIdx.x % p.n_groups) + p.n_groups - 1) / p.n_groups;
  const int n = (int)(pl.end - pl.begin) * rounds;
  if (n == 0) return;  // the whole CTA
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform, also to the compiler: 75 instead of 81 us
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int chunks = 8 * n;
  const int d = p.c.head_dim;
  const uint32_t row_bytes = (uint32_t)d * (k8 ? 1 : 2);
  // K: row r, chunk c of 16 bytes at (r, c ^ 4 (r & 1)): the lanes of two rows and
  // four chunks that read together meet eight banks; here of row g, chunks t
  // (even steps) and 4 + t (odd ones)
  const uint32_t ring = smem_addr(sm.ring[warp][0]);
  constexpr bool kSwap = X::kPerRow > 4;
  const uint32_t k_at[2] = {ring + (uint32_t)(g * X::kRowBytes + 16 * t + (kSwap ? 64 * (g & 1) : 0)),
                            ring + (uint32_t)(g * X::kRowBytes + 16 * t + (kSwap ? 64 - 64 * (g & 1) : 64))};
  // V: chunk c at c ^ (r & 7), of four-chunk rows c ^ (r / 2 & 3); here of rows 2 t
  // and 2 t + 1, this lane group's chunk
  uint32_t v_at[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = 2 * t + u;
    v_at[u] = ring + X::kK + (uint32_t)(r * X::kRowBytes + (X::kPerRow > 4 ? (g ^ r) * 16 : ((g >> 1) ^ (r >> 1)) * 16 + (g & 1) * 8));
  }
  const uint32_t ring_side = ring + X::kK + X::kV;
  const float scale = p.scale * kLog2e;
  const bool guard = p.q.T > 1 || p.q.tree != nullptr;  // rows may hide newest tokens from one another

  // ---- copies of this warp's chunks, kStages ahead: K and V apart, each into
  // the place that its predecessor has just left ----
  const bool pow2 = (p.c.page_size & (p.c.page_size - 1)) == 0;
  const int shift = 31 - __clz(p.c.page_size);
  const bool one_page = p.c.page_size % 16 == 0;  // a chunk never leaves its page
  const int page_step = p.c.n_kv_heads * p.c.page_size;
  // this lane copies the 16-byte pieces lane, lane + 32, ... of the 16 rows
  constexpr int kCopies = 16 * X::kPerRow / 32;
  auto place = [&](int i, bool v) {
    const int r = (32 * i + lane) / X::kPerRow, c = (32 * i + lane) % X::kPerRow;
    const int to = X::kPerRow > 4 ? c ^ (v ? r & 7 : 4 * (r & 1)) : v ? c ^ (r / 2 & 3) : c;
    return ring + (uint32_t)((v ? X::kK : 0) + r * X::kRowBytes + 16 * to);
  };
  // and of the bias, K and V scales four keys of one of them
  const int side_kind = lane >> 2, side_key = 4 * t;
  const float* side_src = side_kind == 0 ? p.c.bias : side_kind == 1 ? p.c.k_scale : side_kind == 2 ? p.c.v_scale : nullptr;
  const unsigned char* const k_src = static_cast<const unsigned char*>(p.c.k);
  const unsigned char* const v_src = static_cast<const unsigned char*>(p.c.v);
  Cursor at;
  at.start(p, pl);
  at.move(p, pl, warp < chunks ? 16 * warp : 0);
  int todo = warp < chunks ? (chunks - warp + NW - 1) / NW : 0, put = 0;  // chunks to copy, stage
  // pages of keys 0 .. 7 and 8 .. 15 of the next chunk, looked up a chunk ahead
  int page_a = -1, page_b = -1, add_a = 0, add_b = 0, left = 0, rel = 0;
  auto look_up = [&]() {
    const int32_t* table = p.q.page_table + (int64_t)at.w.b * p.q.table_stride;
    left = (int)at.w.s.total - at.pos;
    const int64_t behind = at.pos - at.w.s.ctx;
    rel = behind < -64 ? -64 : (int)behind;
    page_a = page_b = -1;
    if (left > 0) {
      const int q = pow2 ? at.pos >> shift : at.pos / p.c.page_size;
      add_a = at.w.hk * p.c.page_size + at.pos - q * p.c.page_size;
      page_a = __ldg(table + q);
    }
    if (!one_page && left > 8) {
      const int pos = at.pos + 8, q = pow2 ? pos >> shift : pos / p.c.page_size;
      add_b = at.w.hk * p.c.page_size + pos - q * p.c.page_size;
      page_b = __ldg(table + q);
    }
  };
  // of the chunk being copied: its rows (the first of either eight) and how many exist
  bool live = false, whole = false;
  int rows[2] = {0, 0}, exist[2] = {0, 0};
  auto copy_rows = [&](uint32_t stage, const unsigned char* src, bool v) {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = (32 * i + lane) / X::kPerRow, c = (32 * i + lane) % X::kPerRow;
      const bool real = (r & 7) < (r < 8 ? exist[0] : exist[1]) && c * X::kE < d;
      copy_async(place(i, v) + stage,
                 src + (real ? (int64_t)((r < 8 ? rows[0] : rows[1]) + (r & 7)) * row_bytes + 16 * c : 0), real ? 16 : 0);
    }
  };
  auto issue_k = [&]() {
    live = todo > 0;
    if (live) {
      const bool in_a = page_a >= 0 && page_a < p.c.n_pages;
      whole = one_page && in_a && left >= 16 && d == kD;
      const uint32_t stage = (uint32_t)put * X::kStage;
      if (whole) {
        rows[0] = page_a * page_step + add_a;
        const unsigned char* k = k_src + (int64_t)rows[0] * X::kRowBytes + 16 * lane;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) copy_async(place(i, false) + stage, k + 512 * i);
        if (side_src)
          copy_async(ring_side + stage + side_kind * 64 + t * 16, side_src + rows[0] + side_key);
        if (lane == 0) sm.info[warp][put] = make_int2(0xffff, rel);  // rel >= -15: newest tokens among them
      } else {
        // the rows that exist; the others become zeros
        const int pb = one_page ? page_a : page_b, ab = one_page ? add_a + 8 : add_b;
        const bool in_b = pb >= 0 && pb < p.c.n_pages;
        exist[0] = in_a ? min(max(left, 0), 8) : 0;
        exist[1] = in_b ? min(max(left - 8, 0), 8) : 0;
        rows[0] = exist[0] ? page_a * page_step + add_a : 0;
        rows[1] = exist[1] ? pb * page_step + ab : 0;
        copy_rows(stage, k_src, false);
        if (side_src) {
          const bool key = (side_key & 7) < (side_key < 8 ? exist[0] : exist[1]);
          copy_async(ring_side + stage + side_kind * 64 + t * 16,
                     side_src + (key ? (side_key < 8 ? rows[0] : rows[1]) + (side_key & 7) : 0), key ? 16 : 0);
        }
        if (lane == 0) sm.info[warp][put] = make_int2((0xff >> (8 - exist[0])) | (0xff >> (8 - exist[1])) << 8, rel);
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  auto issue_v = [&]() {
    if (live) {
      const uint32_t stage = (uint32_t)put * X::kStage;
      if (whole) {
        const unsigned char* v = v_src + (int64_t)rows[0] * X::kRowBytes + 16 * lane;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) copy_async(place(i, true) + stage, v + 512 * i);
      } else {
        copy_rows(stage, v_src, true);
      }
      if (--todo > 0) {
        at.move(p, pl, 16 * NW);
        look_up();
      }
    }
    if (++put == S) put = 0;
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  if (todo > 0) look_up();
#pragma unroll 1
  for (int i = 0; i < S; ++i) {
    issue_k();
    issue_v();
  }

  // ---- pieces ----
  int base = 0, get = 0, mine = warp;  // tiles before the piece, stage, chunk
  for (int rt = blockIdx.x % p.n_groups; rt < p.n_row_tiles; rt += p.n_groups) {
    TreeWalk walk;
    walk.start(p, pl);
    TreePiece w;
    while (walk.next(p, w)) {
      const int stop = 8 * (base + w.k1 - w.k0);
      // queries: row g of each tile, four elements a k step
      uint2 q[X::kQShared ? 1 : kNT][X::kSteps];
      // of rows 2 t and 2 t + 1: what undoes their scaling, times the softmax scale; the token
      float unit[kNT][2];
      int tok[kNT][2];
      if (X::kQShared || mine < stop) {
#pragma unroll
        for (int m = 0; m < kNT; ++m) {
          uint2 (&qm)[X::kSteps] = q[X::kQShared ? 0 : m];
          const TreeRow row = tree_row(p, w.hk, rt, 8 * m + g);
          const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.q.q) + w.b * p.q.q_seq_stride +
                                     row.h * p.q.q_head_stride + row.t * p.q.q_row_stride;
          uint32_t top = 0;
#pragma unroll
          for (int s = 0; s < X::kSteps; ++s) {
            // the chunk of k step s, and the four elements in it
            const int c = s / (X::kE / 4), at4 = (4 * c + t) * X::kE + 4 * (s % (X::kE / 4));
            uint2 v = make_uint2(0u, 0u);
            if (row.exists && at4 < d) v = *reinterpret_cast<const uint2*>(src + at4);
            qm[s] = v;
            top = max(top, max(max((v.x >> 7) & 0xffu, (v.x >> 23) & 0xffu), max((v.y >> 7) & 0xffu, (v.y >> 23) & 0xffu)));
          }
          float undo = scale;
          if constexpr (k8) {
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int up = top == 0 || top == 255 ? 0 : min(14 + 127 - (int)top, 120);
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
            undo = scale * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int s = 0; s < X::kSteps; ++s) {
              const uint2 x = qm[s];
              qm[s].x = pack<true>(__uint_as_float(x.x << 16) * f, __uint_as_float(x.x & 0xffff0000u) * f);
              qm[s].y = pack<true>(__uint_as_float(x.y << 16) * f, __uint_as_float(x.y & 0xffff0000u) * f);
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            unit[m][h] = __shfl_sync(0xffffffffu, undo, 4 * (2 * t + h));
            const TreeRow own = tree_row(p, w.hk, rt, 8 * m + 2 * t + h);
            tok[m][h] = own.exists ? (int)own.t : 0x7fffffff;
          }
          // every warp has the same ones; those of the last piece are no longer read
          if (X::kQShared && warp == m) {
#pragma unroll
            for (int s = 0; s < X::kSteps; ++s) *reinterpret_cast<uint2*>(sm.q + ((m * X::kSteps + s) * 32 + lane) * 8) = qm[s];
          }
        }
      }
      if constexpr (X::kQShared) __syncthreads();
      auto query = [&](int m, int s) {
        if constexpr (X::kQShared) {
          uint32_t a[2];
          load_words<2>(smem_addr(sm.q) + (uint32_t)((m * X::kSteps + s) * 32 + lane) * 8, a);
          return make_uint2(a[0], a[1]);
        } else {
          return q[m][s];
        }
      };
      float o[kNT][X::kTiles][4], mx[kNT][2], l[kNT][2];
#pragma unroll
      for (int m = 0; m < kNT; ++m) {
        mx[m][0] = mx[m][1] = -INFINITY;
        l[m][0] = l[m][1] = 0.f;
#pragma unroll
        for (int j = 0; j < X::kTiles; ++j) o[m][j][0] = o[m][j][1] = o[m][j][2] = o[m][j][3] = 0.f;
      }
      int v_exp = -128;   // exponent of the V scales of this warp's first keys; -128: no keys
      float v_unit = 1.f;
      if constexpr (k8) {
        if (mine < stop) {
          asm volatile("cp.async.wait_group %0;\n" ::"n"(2 * S - 1) : "memory");
          __syncwarp();
          float most = load_one(ring_side + (uint32_t)get * X::kStage + 128 + 4 * (lane & 15));
#pragma unroll
          for (int off = 8; off > 0; off /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
          v_exp = scale_exponent(most);
          v_unit = two_to(kWeightUp - v_exp);
        }
      }
#pragma unroll 1
      for (; mine < stop; mine += NW) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(2 * S - 1) : "memory");  // K and scales of this chunk
        __syncwarp();  // other lanes' scales and info
        const uint32_t from = (uint32_t)get * X::kStage;
        const int2 info = sm.info[warp][get];
        if (++get == S) get = 0;
        // ---- scores: keys g (e < 2) and g + 8, rows 2 t + (e & 1) ----
        float s[kNT][4];
#pragma unroll
        for (int m = 0; m < kNT; ++m) s[m][0] = s[m][1] = s[m][2] = s[m][3] = 0.f;
#pragma unroll
        for (int c = 0; c < X::kKC; ++c) {
          uint32_t kw[2][4];
          load_words<4>(k_at[c & 1] + from + 128 * (c >> 1), kw[0]);
          load_words<4>(k_at[c & 1] + from + 128 * (c >> 1) + 8 * X::kRowBytes, kw[1]);
          constexpr int kPer = X::kE / 4;  // k steps of a chunk
#pragma unroll
          for (int x = 0; x < kPer; ++x) {
            uint32_t a[4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if constexpr (k8) {
                widen_word<kMode>(kw[u][x], a[u], a[2 + u]);
              } else {
                a[u] = kw[u][2 * x];
                a[2 + u] = kw[u][2 * x + 1];
              }
            }
#pragma unroll
            for (int m = 0; m < kNT; ++m) {
              const uint2 b = query(m, kPer * c + x);
              mma<k8>(s[m], a, b.x, b.y);
            }
          }
        }
        // ---- scale, bias, mask, weights ----
        float bias[2] = {0.f, 0.f}, ks[2], vs[2];
        bool all = info.x == 0xffff && info.y + 15 < 0;
        if (p.c.bias) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            bias[u] = load_one(ring_side + from + 32 * u + 4 * g);
            if (bias[u] > -INFINITY && bias[u] < INFINITY) bias[u] = fminf(fmaxf(bias[u] * kLog2e, -kMost), kMost);
          }
          all = all && !__any_sync(0xffffffffu, bias[0] == -INFINITY || bias[1] == -INFINITY);
        }
        if constexpr (k8) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            ks[u] = load_one(ring_side + from + 64 + 32 * u + 4 * g);
            vs[u] = load_one(ring_side + from + 128 + 32 * u + 4 * g) * v_unit;
            vs[u] = vs[u] < kLeastScale ? kLeastScale : vs[u];
            if (p.c.bias && fabsf(bias[u]) >= kHuge) vs[u] = vs[u] > kMostHuge ? kMostHuge : vs[u];
          }
        }
        uint32_t pr[kNT][2];
        // `hidden`: some row does not see some key; see[m], bit e, says which
        uint32_t see[kNT], broken = 0;
        auto weights = [&](auto hidden) {
          constexpr bool kHidden = decltype(hidden)::value;
#pragma unroll
          for (int m = 0; m < kNT; ++m) {
            auto seen = [&](int e) { return !kHidden || ((see[m] >> e) & 1); };
            // weights from the scores and the running max; true when one is too large
            float w4[4], raw[4];
            auto weigh = [&]() {
              bool over = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float y = exp2_approx(s[m][e] - mx[m][e & 1]);
                if (kHidden) y = seen(e) ? y : 0.f;
                raw[e] = y;
                if constexpr (k8) {
                  y *= vs[e >> 1];
                  if (kHidden) y = seen(e) ? y : 0.f;  // a hidden key's scale may be NaN
                }
                w4[e] = y;
                over = over || y > (k8 ? 256.f * (1 << kWeightUp) : 256.f);
              }
              return over;
            };
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = s[m][e] * unit[m][e & 1];
              if constexpr (k8) x = fmaf(x, ks[e >> 1], bias[e >> 1]);
              else x += bias[e >> 1];
              if (kHidden && ((broken >> (g + 8 * (e >> 1))) & 1)) x = __uint_as_float(0x7fc00000u);
              s[m][e] = x;
            }
            if (__any_sync(0xffffffffu, weigh())) {
              // move the max of the rows to the largest score (with its V scale) so far, rescale
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float top = mx[m][h];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  float x = s[m][2 * u + h];
                  // (a NaN scale is not to move the max: it makes the row NaN by its product)
                  if constexpr (k8)
                    if (fabsf(x) < kHuge) x += log2f(fminf(fmaxf(vs[u], kLeastScale), kMostScale)) - kWeightUp;
                  if (seen(2 * u + h)) top = fmaxf(top, x);
                }
#pragma unroll
                for (int off = 4; off < 32; off *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                const float f = top == mx[m][h] ? 1.f : exp2f(mx[m][h] - top);
                mx[m][h] = top;
                l[m][h] *= f;
#pragma unroll
                for (int j = 0; j < X::kTiles; ++j) {
                  o[m][j][h] *= f;
                  o[m][j][2 + h] *= f;
                }
              }
              weigh();
            }
            l[m][0] += raw[0] + raw[2];
            l[m][1] += raw[1] + raw[3];
            pr[m][0] = transpose(pack<k8>(w4[0], w4[1]));
            pr[m][1] = transpose(pack<k8>(w4[2], w4[3]));
          }
        };
        if (all) {
          weights(std::false_type{});
        } else {
          if (kMode != DCC_KV_INT8 && info.y + 15 >= 0 && guard) {
            // newest values that are not finite become zeros -- a row that does
            // not see them must not get 0 * inf --, and the rows that do, NaN
            // (e4m3: the NaN code, which a pool may hold that was filled elsewhere)
            asm volatile("cp.async.wait_group %0;\n" ::"n"(2 * S - 2) : "memory");  // V of this chunk
            __syncwarp();
#pragma unroll 1
            for (int u = 0; u < 4; ++u) {
              const int key = 2 * t + (u & 1) + 8 * (u >> 1);
              if (info.y + key < 0) continue;
              for (int c = 0; c < X::kVC; ++c) {
                const uint32_t a = v_at[u & 1] + from + (u >> 1) * 8 * X::kRowBytes + 128 * c;
                constexpr int kWords = X::kVB / 4;
                uint32_t x[kWords];
                load_words<kWords>(a, x);
                const uint32_t was = broken;
#pragma unroll
                for (int e = 0; e < kWords; ++e) {
                  if constexpr (k8) {
                    const uint32_t nan = (((x[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;  // 1 in the bytes of 0x7f, 0xff
                    if (nan) x[e] &= ~(nan * 255u), broken |= 1u << key;
                  } else {
                    if ((x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u, broken |= 1u << key;
                    if ((x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0x0000ffffu, broken |= 1u << key;
                  }
                }
                if (broken != was) store_words<kWords>(a, x);
              }
            }
            broken = __reduce_or_sync(0xffffffffu, broken);
          }
#pragma unroll
          for (int m = 0; m < kNT; ++m) see[m] = 0;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int key = g + 8 * u, i = info.y + key;
            if (((info.x >> key) & 1) && bias[u] != -INFINITY && i < w.s.cnt) {
#pragma unroll
              for (int m = 0; m < kNT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if (i < 0 || (tok[m][h] < p.q.T && tree_sees(p, w.b, tok[m][h], i))) see[m] |= 1u << (2 * u + h);
            }
          }
          __syncwarp();
          weights(std::true_type{});
        }
        __syncwarp();  // the scales and info have been read
        issue_k();
        // ---- values ----
        asm volatile("cp.async.wait_group %0;\n" ::"n"(2 * S - 1) : "memory");
        __syncwarp();
#pragma unroll
        for (int c = 0; c < X::kVC; ++c) {
          uint32_t vw[4][X::kVB / 4];
#pragma unroll
          for (int u = 0; u < 4; ++u) load_words<X::kVB / 4>(v_at[u & 1] + from + (u >> 1) * 8 * X::kRowBytes + 128 * c, vw[u]);
#pragma unroll
          for (int x = 0; x < X::kVB / 4; ++x) {
            if constexpr (k8) {
#pragma unroll
              for (int y = 0; y < 4; y += 2) {
                const uint32_t a[4] = {join_codes<kMode>(vw[0][x], vw[1][x], y), join_codes<kMode>(vw[0][x], vw[1][x], y + 1),
                                       join_codes<kMode>(vw[2][x], vw[3][x], y), join_codes<kMode>(vw[2][x], vw[3][x], y + 1)};
#pragma unroll
                for (int m = 0; m < kNT; ++m) mma<true>(o[m][2 * x + y / 2], a, pr[m][0], pr[m][1]);
              }
            } else {
              const uint32_t a[4] = {__byte_perm(vw[0][x], vw[1][x], 0x5410), __byte_perm(vw[0][x], vw[1][x], 0x7632),
                                     __byte_perm(vw[2][x], vw[3][x], 0x5410), __byte_perm(vw[2][x], vw[3][x], 0x7632)};
#pragma unroll
              for (int m = 0; m < kNT; ++m) mma<false>(o[m][4 * c + x], a, pr[m][0], pr[m][1]);
            }
          }
        }
        __syncwarp();
        issue_v();
      }

      // ---- the piece is done: warps together, two rows at a time ----
#pragma unroll
      for (int m = 0; m < kNT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int off = 4; off < 32; off *= 2) l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], off);
          if (g == 0) {
            sm.m[warp][8 * m + 2 * t + h] = mx[m][h];
            sm.l[warp][8 * m + 2 * t + h] = l[m][h];
          }
        }
      if (lane == 0) sm.up[warp] = v_exp;
      __syncthreads();
      int most_up = 0;
      float to_most = 1.f, from_most = 1.f;  // from this warp's units to those of the largest, from those to none
      if constexpr (k8) {
        most_up = sm.up[0];
#pragma unroll
        for (int x = 1; x < NW; ++x) most_up = max(most_up, sm.up[x]);
        to_most = two_to(max(v_exp - most_up - kWeightUp, -126));
        from_most = two_to(most_up);
      }
      const int64_t rows_left = p.q.T * p.group - (int64_t)rt * kRows;
      const int rows = rows_left < kRows ? (int)rows_left : kRows;
#pragma unroll
      for (int m = 0; m < kNT; ++m)
#pragma unroll 1
        for (int r0 = 8 * m; r0 < min(rows, 8 * m + 8); r0 += 2) {
          if (2 * t == (r0 & 7)) {  // this lane has the two rows
            float f[2];
            bool none[2];  // a warp that saw no key of the row has nothing to add
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float top = -INFINITY;
              for (int x = 0; x < NW; ++x) top = fmaxf(top, sm.m[x][r0 + h]);
              const float own = sm.m[warp][r0 + h];
              none[h] = sm.l[warp][r0 + h] == 0.f;
              f[h] = (own == top ? 1.f : exp2f(own - top)) * to_most;  // 0 is a factor too: O may hold a NaN
            }
            float* dst = sm.sum + warp * 2 * kD;
#pragma unroll
            for (int j = 0; j < X::kTiles; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int col = (k8 ? X::kVB * g + 2 * j : (j >> 2) * 64 + 8 * g + 2 * (j & 3)) + (e >> 1);
                dst[(e & 1) * kD + col] = none[e & 1] ? 0.f : f[e & 1] * o[m][j][e];
              }
          }
          __syncthreads();
          for (int i = threadIdx.x; i < 2 * kD; i += X::kThreads) {
            const int r = r0 + i / kD, col = i % kD;
            float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
            for (int x = 0; x < NW; ++x) top = fmaxf(top, sm.m[x][r]);
#pragma unroll
            for (int x = 0; x < NW; ++x) {
              const float lx = sm.l[x][r];
              if (lx != 0.f) sum = fmaf(sm.m[x][r] == top ? 1.f : exp2f(sm.m[x][r] - top), lx, sum);
              acc += sm.sum[x * 2 * kD + i];
            }
            // -kMost: nothing but biases of the type's lowest value
            const float ln = top == -kMost ? -kMost : top * kLn2;
            const TreeRow row = tree_row(p, w.hk, rt, r);
            if (r >= rows) continue;
            if (row.t >= w.s.cnt) sum = 0.f;  // a row that does not exist
            const float out = sum != 0.f ? acc / sum * from_most : 0.f;
            if (w.part >= 0) {
              const int64_t part = p.part_row(span, rt, w.part, r);
              if (col < d) p.part_o[part * kTreePartCols + col] = out;
              if (col == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(ln, sum);
            } else {
              if (col < d) tree_out_row<__nv_bfloat16>(p, w.b, row)[col] = __float2bfloat16_rn(out);
              if (col == 0 && p.q.lse)
                p.q.lse[((int64_t)w.b * p.q.n_q_heads + row.h) * p.q.T + row.t] = sum != 0.f ? ln + logf(sum) : -INFINITY;
            }
          }
          __syncthreads();
        }
      base += w.k1 - w.k0;
    }
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");
}

template <int kMode, int kD, int kNT>
static int launch(const TreeParams& p, cudaStream_t st) {
  using X = Shape<kMode, kD, kNT>;
  constexpr size_t smem = sizeof(Smem<X, kNT>);
  static_assert(smem <= kSmemLimit, "shared memory");
  auto kernel = tree_mma_kernel<kMode, kD, kNT>;
  DCC_CHECK(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "tree_mma smem"));
  kernel<<<p.n_groups * p.n_spans, X::kThreads, smem, st>>>(p);
  return check_launch("tree_attention");
}
template <int kMode, int kD>
static int launch_n(const TreeParams& p, cudaStream_t st) {
  return p.n_rows == 8 ? launch<kMode, kD, 1>(p, st) : launch<kMode, kD, 2>(p, st);
}
template <int kMode>
static int launch_d(const TreeParams& p, cudaStream_t st) {
  return p.c.head_dim <= 64 ? launch_n<kMode, 64>(p, st) : launch_n<kMode, 128>(p, st);
}

}  // namespace tm

int launch_tree_mma(const TreeParams& p, cudaStream_t st) {
  switch (p.c.format) {
    case DCC_KV_INT8: return tm::launch_d<DCC_KV_INT8>(p, st);
    case DCC_KV_E4M3: return tm::launch_d<DCC_KV_E4M3>(p, st);
    default: return tm::launch_d<DCC_KV_BF16>(p, st);
  }
}

}  // namespace dcc
