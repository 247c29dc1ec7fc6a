// Work of the tree attention and its division among CTAs.
//
// The rows of one sequence and KV head -- T newest tokens x `group` query
// heads, row = t * group + g -- are cut into tiles of `n_rows`, its cached
// tokens into tiles of 128 keys.  The key tiles of all (sequence, KV head), in
// that order, form one line that is cut into n_spans equal spans (+-1 tile; one
// tile each where there are fewer tiles), whatever the lengths.  CTA
// (span, group) walks over its span for the row tiles group, group + n_groups,
// ...: the CTAs that read the same keys for other rows are neighbours and run
// at the same time, so the keys come from HBM once.  A (sequence, KV head) that
// does not lie in one span leaves partial results (output, max, sum),
// which tree_merge_kernel adds in the order of the spans -- no atomics, so
// results repeat bit for bit.  The lengths are read on the device: neither the
// launch nor a captured graph depends on them.
#pragma once

#include "kv_pages.cuh"

namespace dcc {

constexpr int kTreeKeys = 128;
constexpr int kTreePartCols = 128;
constexpr int64_t kTreeMaxT = 4096;

struct TreeParams {
  dcc_kv_pages c;
  dcc_tree_query q;
  int group;    // query heads per KV head
  int n_rows;   // rows per row tile
  int n_row_tiles;
  int n_groups, n_spans;
  float scale;
  float* part_o;   // [n_spans][n_row_tiles][2][n_rows][kTreePartCols]
  float* part_ml;  // [n_spans][n_row_tiles][2][n_rows][2]: max, sum

  __host__ __device__ int64_t part_row(int span, int rt, int which, int r) const {
    return (((int64_t)span * n_row_tiles + rt) * 2 + which) * n_rows + r;
  }
};

struct SeqTokens {
  int64_t ctx;    // positions before the newest
  int64_t total;  // positions that are looked at (0 when no row asks)
  int cnt;        // newest tokens
};
__device__ __forceinline__ SeqTokens tree_tokens(const TreeParams& p, int b) {
  SeqTokens s;
  s.ctx = max(p.q.context[b], 0);
  const int64_t T = p.q.T;
  s.cnt = (int)(p.q.counts ? min(max((int64_t)p.q.counts[b], (int64_t)0), T) : T);
  const int64_t cap = (int64_t)p.q.max_pages * p.c.page_size;
  s.total = s.cnt > 0 ? min(s.ctx + s.cnt, cap) : 0;
  return s;
}
__device__ __forceinline__ int64_t tree_key_tiles(const SeqTokens& s) { return (s.total + kTreeKeys - 1) / kTreeKeys; }

__device__ __forceinline__ bool tree_sees(const TreeParams& p, int b, int64_t t, int64_t i) {
  return p.q.tree ? p.q.tree[b * p.q.tree_seq_stride + t * p.q.T + i] != 0 : i <= t;
}

// Where weights are held in fp16 (beside 8-bit codes) they carry the V scale, in
// units of 2^(e - 6) with e the exponent of the largest V scale of the first
// keys of a part (0 where those have none): the first weights are below 2^7
// whatever the values' size, and six bits more of small weights are kept.  2^8
// on, where the running max has to move, fp16 still reaches.  (Scales of one
// sequence that differ by more than 2^90 are beyond this.)
// Scores beyond kHuge, biases of a mask, do not hold a logarithm added to them (a
// row of zeros has the scale 2^-96: -1e9 - 96 is -1e9 - 128 in fp32, and the weight
// 2^128): there the max is taken of the scores alone, and of such a key's V scale
// no more than kMostHuge counts, so that rows which see nothing else stay finite.
constexpr int kWeightUp = 6;
constexpr float kHuge = 16777216.f, kMostHuge = 8192.f;
constexpr float kLeastScale = 5.048709793e-29f;  // 2^-94, in those units: rows that were never written have scale 0
constexpr float kMostScale = 3.402823466e38f;
__device__ __forceinline__ int scale_exponent(float largest) {
  const int e = (int)(__float_as_uint(largest) >> 23) - 127;
  return e < -64 || e > 126 ? 0 : e;  // rows of zeros or never written, or not a number
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// n spans of `total` >= n tiles, none empty.
__device__ __forceinline__ int span_count(int64_t total, int n_spans) { return (int)(total < n_spans ? total : n_spans); }
__device__ __forceinline__ int64_t span_begin(int64_t total, int i, int n) { return total * i / n; }
// The span that holds tile g.
__device__ __forceinline__ int span_owner(int64_t total, int64_t g, int n) { return (int)(((g + 1) * n - 1) / total); }

// Where a span begins: the sequence that holds tile `begin` and the number of
// its first tile.
struct TreePlan {
  int64_t total, begin, end, seq_off;
  int seq;
};
struct TreePlanSmem {
  int64_t warp[32];
  TreePlan plan;
};
// All threads of the block; ends with a __syncthreads.
__device__ __forceinline__ void tree_plan(const TreeParams& p, int span, TreePlanSmem& sm) {
  const int n_thr = blockDim.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n_warps = (n_thr + 31) >> 5;
  const int64_t heads = p.c.n_kv_heads;
  int64_t sum = 0;
  for (int b = tid; b < p.q.n_seqs; b += n_thr) sum += heads * tree_key_tiles(tree_tokens(p, b));
  sum = warp_sum(sum);
  if (lane == 0) sm.warp[warp] = sum;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < n_warps; ++w) total += sm.warp[w];
  const int n = span_count(total, p.n_spans);
  const int64_t begin = span < n ? span_begin(total, span, n) : 0, end = span < n ? span_begin(total, span + 1, n) : 0;
  if (tid == 0) sm.plan = TreePlan{total, begin, end, 0, 0};
  if (begin < end) {  // the same for every thread
    int64_t carry = 0;
    for (int b0 = 0; b0 < p.q.n_seqs && carry <= begin; b0 += n_thr) {
      const int b = b0 + tid;
      const int64_t w = b < p.q.n_seqs ? heads * tree_key_tiles(tree_tokens(p, b)) : 0;
      int64_t incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      __syncthreads();
      if (lane == 31) sm.warp[warp] = incl;
      __syncthreads();
      int64_t before = carry;
      for (int i = 0; i < n_warps; ++i) {
        if (i < warp) before += sm.warp[i];
        carry += sm.warp[i];
      }
      const int64_t off = before + incl - w;
      if (off <= begin && begin < off + w) {
        sm.plan.seq = b;
        sm.plan.seq_off = off;
      }
    }
  }
  __syncthreads();
}

// The pieces of a span, one (sequence, KV head) or the part of it in the span
// after the other.  Every role of a CTA walks the same pieces.
struct TreePiece {
  int b, hk;
  int k0, k1;  // key tiles
  SeqTokens s;
  int part;    // -1: all keys, else the partial slot (0: begun by an earlier span, 1: begun here)
};
struct TreeWalk {
  int64_t g, end, off;  // next tile, end of span, first tile of sequence b
  int tiles, b;         // key tiles of b
  SeqTokens s;
  __device__ __forceinline__ void start(const TreeParams& p, const TreePlan& pl) {
    g = pl.begin;
    end = pl.end;
    off = pl.seq_off;
    b = pl.seq;
    tiles = 0;
    if (g < end) {
      s = tree_tokens(p, b);
      tiles = (int)tree_key_tiles(s);
    }
  }
  __device__ __forceinline__ bool next(const TreeParams& p, TreePiece& o) {
    if (g >= end) return false;
    while (g >= off + (int64_t)p.c.n_kv_heads * tiles) {  // ends: g < end <= the tiles of all sequences
      off += (int64_t)p.c.n_kv_heads * tiles;
      s = tree_tokens(p, ++b);
      tiles = (int)tree_key_tiles(s);
    }
    const int64_t in_seq = g - off;
    o.hk = (int)(in_seq / tiles);
    o.k0 = (int)(in_seq - (int64_t)o.hk * tiles);
    const int64_t left = end - g;
    o.k1 = left < tiles - o.k0 ? o.k0 + (int)left : tiles;
    o.b = b;
    o.s = s;
    o.part = o.k0 > 0 ? 0 : (o.k1 < tiles ? 1 : -1);
    g += o.k1 - o.k0;
    return true;
  }
};

// q row of the tile: token, query head; valid when it exists.
struct TreeRow {
  int64_t t;
  int h;
  bool exists;
};
__device__ __forceinline__ TreeRow tree_row(const TreeParams& p, int hk, int rt, int r) {
  const int row = rt * p.n_rows + r;  // the rows of a KV head are fewer than 2^25
  const int t = row / p.group;
  TreeRow o;
  o.t = t;
  o.h = hk * p.group + row - t * p.group;
  o.exists = o.t < p.q.T;
  return o;
}

template <typename T>
__device__ __forceinline__ T* tree_out_row(const TreeParams& p, int b, const TreeRow& r) {
  return static_cast<T*>(p.q.o) + b * p.q.o_seq_stride + r.h * p.q.o_head_stride + r.t * p.q.o_row_stride;
}

// ---- what both tensor-core kernels are made of ----
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, uint32_t size) {  // 16 bytes; of size < 16 the rest are zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(size) : "memory");
}
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool kHalf>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if constexpr (kHalf) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// int8 code in the low byte of each half, 0x64 above it and its sign flipped:
// the fp16 number 1024 + 128 + code
__device__ __forceinline__ uint32_t less_1152(uint32_t y) {
  const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t from_e4m3(uint32_t two) {
  const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return (uint32_t)r.x | (uint32_t)r.y << 16;
}
// Codes 0, 1 and 2, 3 of a word as two pairs of fp16.
template <int kMode>
__device__ __forceinline__ void widen_word(uint32_t w, uint32_t& b0, uint32_t& b1) {
  if constexpr (kMode == DCC_KV_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    b0 = less_1152(__byte_perm(u, 0x64646464u, 0x4140));
    b1 = less_1152(__byte_perm(u, 0x64646464u, 0x4342));
  } else {
    b0 = from_e4m3(w & 0xffffu);
    b1 = from_e4m3(w >> 16);
  }
}

// The tensor-core kernels: bf16 queries, bf16 or 8-bit cache, head_dim a
// multiple of 16, page_size of 8.  tree_mma.cu for up to 16 rows per KV head,
// tree_tc05.cu for more.
bool tree_tensor_supported(const dcc_kv_pages& c, const dcc_tree_query& q, int dtype);
int launch_tree_mma(const TreeParams& p, cudaStream_t st);
int launch_tree_tc05(const TreeParams& p, cudaStream_t st);

}  // namespace dcc
