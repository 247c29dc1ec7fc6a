// Tree attention over the paged cache for few query rows (up to 32 per KV
// head): bf16 queries, bf16 / int8 / e4m3 cache, head_dim a multiple of 16.
//
// With few rows every key is used for so little arithmetic that HBM is the
// bound, and what a kernel has to save is instructions per key.  Here every
// warp works alone on 16 keys at a time, and a lane copies (cp.async) exactly
// the bytes that it will feed to its own MMA operands, so the shared memory
// ring is private to the lane: no barriers, no swizzle, no second trip through
// shared memory for widened codes.  The contractions are register MMAs
// (m16n8k16, 16 query rows), which are far from their limit:
//   S [16 rows, 8 keys]  += Q K^T    the k index runs over d in the order in
//                                    which a lane's 16-byte chunks hold it
//   O [16 rows, 8 cols]  += P V      column n of n-tile j stands for the
//                                    element of V that lane group n holds as
//                                    its j-th, so pairs of keys are joined by
//                                    byte permutes and never transposed
// Codes become fp16, exactly; scales act on S and P in fp32.  Beside them the
// queries are held in fp16 too, each row scaled by a power of two that takes
// its largest element to 2^14: bf16 digits fit, and what falls below fp16's
// range is under 2^-39 of that element.
// Each warp keeps a running max that moves when a score passes it by 2^8, its
// sums and O in registers; the warps are added up at the end of a piece.  P is
// rounded once, to bf16 beside bf16 values (a relative 2^-9 of each weight), to
// fp16 beside codes (2^-12): there P carries the V scale, so the max is taken
// over score + log2(scale), which keeps P below 2^8 whatever the scales are.
#include <string>

#include "tree_attention.cuh"

namespace dcc {
namespace tm {

constexpr size_t kSmemLimit = 232448;

template <int kMode, int kD, int kMT>  // cache format, padded head_dim, 16-row tiles
struct Shape {
  static constexpr bool k8 = kMode != DCC_KV_BF16;
  // as many warps as the registers of a warp allow (and the ring has to hold
  // 64 KB and more in flight)
  static constexpr int kWarps = k8 && kMT == 1 ? 12 : 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kE = k8 ? 16 : 8;             // elements of a 16-byte chunk
  static constexpr int kKC = kD / (4 * kE);          // K chunks of a lane and key
  static constexpr int kVC = k8 ? 1 : kD / 64;       // V chunks of a lane and key
  static constexpr int kVB = k8 ? kD / 8 : 16;       // bytes of one
  static constexpr int kSteps = kD / 16;             // k steps of S
  static constexpr int kTiles = kD / 8;              // n-tiles of O
  static constexpr int kK = 32 * 2 * kKC * 16, kV = 32 * 4 * kVC * kVB, kSide = 3 * 64;
  static constexpr int kStage = kK + kV + kSide;     // 16 keys of a warp
  // operands of the queries: in registers, or, where O takes those, in shared memory
  static constexpr bool kQShared = k8 || kMT == 2;
  static constexpr int kQ = kQShared ? kMT * kSteps * 512 : 16;
  static constexpr int kSum = kWarps * 2 * kD * 4;   // O of two rows of every warp
  static constexpr size_t kFixed = kSum + (size_t)kWarps * 16 * kMT * 8 + kWarps * 64 + kQ + 1024;
  static constexpr int kFit = (int)((kSmemLimit - kFixed) / ((size_t)kStage * kWarps));
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static_assert(kStages >= 2, "ring");
};

template <typename X, int kMT>
struct Smem {
  unsigned char ring[X::kWarps][X::kStages][X::kStage];
  float sum[X::kSum / 4];
  __align__(16) unsigned char q[X::kQ];
  float m[X::kWarps][16 * kMT], l[X::kWarps][16 * kMT];
  int2 info[X::kWarps][X::kStages];  // keys that exist (16 bits), first key behind the context
  TreePlanSmem plan;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool real) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(real ? 8 : 0) : "memory");
}
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t a, uint32_t* w) {
  if constexpr (kWords == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
  else
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "r"(a) : "memory");
}
__device__ __forceinline__ float2 load_pair(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
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

// The tile that a chunk of 16 keys lies in, for chunks that only grow.
struct Cursor {
  TreeWalk walk;
  TreePiece w;
  int rt, first;  // first tile of the piece, counted over the CTA
  __device__ __forceinline__ void start(const TreeParams& p, const TreePlan& pl) {
    rt = blockIdx.x % p.n_groups;
    walk.start(p, pl);
    first = 0;
    walk.next(p, w);
  }
  __device__ __forceinline__ void seek(const TreeParams& p, const TreePlan& pl, int tile) {
    while (tile >= first + w.k1 - w.k0) {
      first += w.k1 - w.k0;
      if (!walk.next(p, w)) {
        rt += p.n_groups;
        walk.start(p, pl);
        walk.next(p, w);
      }
    }
  }
};

template <int kMode, int kD, int kMT>
__global__ void __launch_bounds__(Shape<kMode, kD, kMT>::kThreads, 1) tree_mma_kernel(const __grid_constant__ TreeParams p) {
  using X = Shape<kMode, kD, kMT>;
  constexpr bool k8 = X::k8;
  constexpr int kRows = 16 * kMT, S = X::kStages, NW = X::kWarps;
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kMost = 3.402823466e38f;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Smem<X, kMT>& sm = *reinterpret_cast<Smem<X, kMT>*>(smem_raw);
  const int span = blockIdx.x / p.n_groups;
  tree_plan(p, span, sm.plan);
  const TreePlan pl = sm.plan.plan;
  const int rounds = (p.n_row_tiles - (int)(blockIdx.x % p.n_groups) + p.n_groups - 1) / p.n_groups;
  const int n = (int)(pl.end - pl.begin) * rounds;
  if (n == 0) return;  // the whole CTA
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int chunks = 8 * n;
  const int d = p.c.head_dim;
  const uint32_t row_bytes = (uint32_t)d * (k8 ? 1 : 2);
  const uint32_t ring = smem_addr(sm.ring[warp][0]) + (uint32_t)lane * 16;
  const uint32_t ring_v = smem_addr(sm.ring[warp][0]) + X::kK + (uint32_t)lane * X::kVB;
  const uint32_t ring_side = smem_addr(sm.ring[warp][0]) + X::kK + X::kV;
  const float scale = p.scale * kLog2e;
  const bool guard = p.q.T > 1 || p.q.tree != nullptr;  // rows may hide newest tokens from one another

  // ---- copies of this warp's chunks, kStages - 1 ahead ----
  Cursor at;
  at.start(p, pl);
  const bool pow2 = (p.c.page_size & (p.c.page_size - 1)) == 0;
  const int shift = 31 - __clz(p.c.page_size);
  const int page_step = p.c.n_kv_heads * p.c.page_size;
  int next = warp, put = 0;  // chunk, stage
  // pages of keys 0 .. 7 and 8 .. 15 of the next chunk, looked up a chunk ahead
  int page[2] = {-1, -1}, add[2] = {0, 0}, left = 0, rel = 0;
  auto look_up = [&]() {
    if (next >= chunks) return;
    at.seek(p, pl, next >> 3);
    const int pos = (at.w.k0 + (next >> 3) - at.first) * kTreeKeys + 16 * (next & 7);
    left = (int)min(at.w.s.total - pos, (int64_t)16);
    const int64_t behind = pos - at.w.s.ctx;
    rel = (int)(behind < -64 ? -64 : behind);
    const int32_t* table = p.q.page_table + (int64_t)at.w.b * p.q.table_stride;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      page[h] = -1;
      if (left > 8 * h) {
        const int q = pos + 8 * h, s = pow2 ? q >> shift : q / p.c.page_size;
        add[h] = at.w.hk * p.c.page_size + q - s * p.c.page_size;
        page[h] = __ldg(table + s);
      }
    }
  };
  auto issue = [&]() {
    if (next < chunks) {
      const bool okA = page[0] >= 0 && page[0] < p.c.n_pages, okB = page[1] >= 0 && page[1] < p.c.n_pages;
      const int nA = okA ? min(max(left, 0), 8) : 0, nB = okB ? min(max(left - 8, 0), 8) : 0;
      const int rowA = nA ? page[0] * page_step + add[0] : 0, rowB = nB ? page[1] * page_step + add[1] : 0;
      const uint32_t to = (uint32_t)put * X::kStage;
      const unsigned char* k = static_cast<const unsigned char*>(p.c.k);
      const unsigned char* v = static_cast<const unsigned char*>(p.c.v);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool key = g < (u ? nB : nA);
        const unsigned char* src = k + (int64_t)(u ? rowB : rowA) * row_bytes + (key ? (uint32_t)g * row_bytes + 16u * t : 0u);
#pragma unroll
        for (int c = 0; c < X::kKC; ++c) {
          const bool real = key && (4 * c + t) * X::kE < d;
          copy_async<16>(ring + to + (u * X::kKC + c) * 512, real ? src + 64 * c : k, real);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
        const int i = 2 * t + (u & 1);
        const bool key = i < (u >> 1 ? nB : nA);
        const unsigned char* src = v + (int64_t)(u >> 1 ? rowB : rowA) * row_bytes + (key ? (uint32_t)i * row_bytes + (uint32_t)(X::kVB * g) : 0u);
#pragma unroll
        for (int c = 0; c < X::kVC; ++c) {
          const bool real = key && X::kVB * g + 128 * c < (int)row_bytes;
          copy_async<X::kVB>(ring_v + to + (u * X::kVC + c) * 32 * X::kVB, real ? src + 128 * c : v, real);
        }
      }
      // bias, K and V scales of the 16 keys, four a lane
      if (k8 || p.c.bias) {
        const int a = lane >> 2, four = 4 * t;
        const float* from = a == 0 ? p.c.bias : a == 1 ? p.c.k_scale : p.c.v_scale;
        if (a < 3 && from) {
          const bool real = (four & 7) < (four < 8 ? nA : nB);
          copy_async<16>(ring_side + to + a * 64 + t * 16, real ? from + (four < 8 ? rowA + four : rowB + four - 8) : from, real);
        }
      }
      if (lane == 0) sm.info[warp][put] = make_int2((0xff >> (8 - nA)) | (0xff >> (8 - nB)) << 8, rel);
      next += NW;
      look_up();
    }
    if (++put == S) put = 0;
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  look_up();
#pragma unroll 1
  for (int i = 0; i < S - 1; ++i) issue();

  // ---- pieces ----
  int base = 0, get = 0, mine = warp;  // tiles before the piece, stage, chunk
  for (int rt = blockIdx.x % p.n_groups; rt < p.n_row_tiles; rt += p.n_groups) {
    TreeWalk walk;
    walk.start(p, pl);
    TreePiece w;
    while (walk.next(p, w)) {
      const int stop = 8 * (base + w.k1 - w.k0);
      // queries: rows g and g + 8 of each 16-row tile, four elements a k step
      uint32_t q[X::kQShared ? 1 : kMT][X::kSteps][4];
      float unit[kMT][2];  // what undoes their scaling, times the softmax scale
      int tok[kMT][2];
      if (X::kQShared || mine < stop) {
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          uint32_t (&qm)[X::kSteps][4] = q[X::kQShared ? 0 : m];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const TreeRow row = tree_row(p, w.hk, rt, 16 * m + 8 * h + g);
            tok[m][h] = row.exists ? (int)row.t : 0x7fffffff;
            const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.q.q) + w.b * p.q.q_seq_stride +
                                       row.h * p.q.q_head_stride + row.t * p.q.q_row_stride;
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < X::kSteps; ++s) {
              // the chunk of k step s, and the four elements in it
              const int c = s / (X::kE / 4), at4 = (4 * c + t) * X::kE + 4 * (s % (X::kE / 4));
              uint2 v = make_uint2(0u, 0u);
              if (row.exists && at4 < d) v = *reinterpret_cast<const uint2*>(src + at4);
              qm[s][h] = v.x;
              qm[s][2 + h] = v.y;
              top = max(top, max(max((v.x >> 7) & 0xffu, (v.x >> 23) & 0xffu), max((v.y >> 7) & 0xffu, (v.y >> 23) & 0xffu)));
            }
            unit[m][h] = scale;
            if constexpr (k8) {
              top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
              top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
              const int up = top == 0 || top == 255 ? 0 : min(14 + 127 - (int)top, 120);
              const float f = __uint_as_float((uint32_t)(127 + up) << 23);
              unit[m][h] = scale * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
              for (int s = 0; s < X::kSteps; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t x = qm[s][2 * e + h];
                  qm[s][2 * e + h] = pack<true>(__uint_as_float(x << 16) * f, __uint_as_float(x & 0xffff0000u) * f);
                }
            }
          }
          // every warp has the same ones; those of the last piece are no longer read
          if (X::kQShared && warp == m % NW) {
#pragma unroll
            for (int s = 0; s < X::kSteps; ++s)
              *reinterpret_cast<uint4*>(sm.q + ((m * X::kSteps + s) * 32 + lane) * 16) = make_uint4(qm[s][0], qm[s][1], qm[s][2], qm[s][3]);
          }
        }
      }
      if constexpr (X::kQShared) __syncthreads();
      auto query = [&](int m, int s, uint32_t* a) {
        if constexpr (X::kQShared) {
          load_words<4>(smem_addr(sm.q) + (uint32_t)((m * X::kSteps + s) * 32 + lane) * 16, a);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = q[m][s][e];
        }
      };
      float o[kMT][X::kTiles][4], mx[kMT][2], l[kMT][2];
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        mx[m][0] = mx[m][1] = -INFINITY;
        l[m][0] = l[m][1] = 0.f;
#pragma unroll
        for (int j = 0; j < X::kTiles; ++j) o[m][j][0] = o[m][j][1] = o[m][j][2] = o[m][j][3] = 0.f;
      }
#pragma unroll 1
      for (; mine < stop; mine += NW) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(S - 2) : "memory");
        __syncwarp();  // the scales and info of the chunk; and the last chunk's have been read
        issue();
        const uint32_t from = (uint32_t)get * X::kStage;
        const int2 info = sm.info[warp][get];
        if (++get == S) get = 0;
        // ---- scores ----
        float s[kMT][2][4];
#pragma unroll
        for (int m = 0; m < kMT; ++m)
#pragma unroll
          for (int u = 0; u < 2; ++u) s[m][u][0] = s[m][u][1] = s[m][u][2] = s[m][u][3] = 0.f;
#pragma unroll
        for (int c = 0; c < X::kKC; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t kw[4];
            load_words<4>(ring + from + (u * X::kKC + c) * 512, kw);
            if constexpr (k8) {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                uint32_t b0, b1;
                widen_word<kMode>(kw[x], b0, b1);
#pragma unroll
                for (int m = 0; m < kMT; ++m) {
                  uint32_t a[4];
                  query(m, 4 * c + x, a);
                  mma<true>(s[m][u], a, b0, b1);
                }
              }
            } else {
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int m = 0; m < kMT; ++m) {
                  uint32_t a[4];
                  query(m, 2 * c + x, a);
                  mma<false>(s[m][u], a, kw[2 * x], kw[2 * x + 1]);
                }
            }
          }
        // ---- scale, bias, mask ----
        float2 bias[2], ks[2], vs[2], lift[2];
        uint32_t broken = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          bias[u] = make_float2(0.f, 0.f);
          lift[u] = make_float2(0.f, 0.f);
          if (p.c.bias) {
            bias[u] = load_pair(ring_side + from + 32 * u + 8 * t);
            if (bias[u].x > -INFINITY && bias[u].x < INFINITY) bias[u].x = fminf(fmaxf(bias[u].x * kLog2e, -kMost), kMost);
            if (bias[u].y > -INFINITY && bias[u].y < INFINITY) bias[u].y = fminf(fmaxf(bias[u].y * kLog2e, -kMost), kMost);
          }
          if constexpr (k8) {
            ks[u] = load_pair(ring_side + from + 64 + 32 * u + 8 * t);
            vs[u] = load_pair(ring_side + from + 128 + 32 * u + 8 * t);
            // from 2^-100: rows that were never written have scale 0
            lift[u].x = __log2f(fmaxf(vs[u].x, 7.888609e-31f));
            lift[u].y = __log2f(fmaxf(vs[u].y, 7.888609e-31f));
          }
        }
        const bool newest = info.y + 15 >= 0;
        uint32_t see[kMT];  // bit 4 u + e of s[u][e]
#pragma unroll
        for (int m = 0; m < kMT; ++m) see[m] = 0xffu;
        bool all = info.x == 0xffff && !newest;
        if (p.c.bias) {
          bool hidden = bias[0].x == -INFINITY || bias[0].y == -INFINITY || bias[1].x == -INFINITY || bias[1].y == -INFINITY;
          all = all && !__any_sync(0xffffffffu, hidden);
        }
        if (!all) {
          if (!k8 && newest && guard) {
            // newest values that are not finite become zeros -- a row that does
            // not see them must not get 0 * inf --, and the rows that do, NaN
#pragma unroll 1
            for (int u = 0; u < 4; ++u) {
              if (info.y + 2 * t + (u & 1) + 8 * (u >> 1) < 0) continue;
              for (int c = 0; c < X::kVC; ++c) {
                const uint32_t a = ring_v + from + (u * X::kVC + c) * 32 * X::kVB;
                uint32_t x[4];
                load_words<4>(a, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if ((x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u, broken |= 1u << u;
                  if ((x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0x0000ffffu, broken |= 1u << u;
                }
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(a), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                             : "memory");
              }
            }
#pragma unroll
            for (int off = 4; off < 32; off *= 2) broken |= __shfl_xor_sync(0xffffffffu, broken, off);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = 2 * t + e + 8 * u, i = info.y + key;
              const float b = e ? bias[u].y : bias[u].x;
              const bool exists = ((info.x >> key) & 1) && b != -INFINITY && i < w.s.cnt;
#pragma unroll
              for (int m = 0; m < kMT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if (!(exists && (i < 0 || (tok[m][h] < p.q.T && tree_sees(p, w.b, tok[m][h], i)))))
                    see[m] &= ~(1u << (4 * u + 2 * h + e));
            }
        }
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          bool over = false;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = s[m][u][e] * unit[m][e >> 1];
              const float b = e & 1 ? bias[u].y : bias[u].x;
              if constexpr (k8) x = fmaf(x, e & 1 ? ks[u].y : ks[u].x, b);
              else x += b;
              if (!all && ((broken >> (2 * u + (e & 1))) & 1)) x = __uint_as_float(0x7fc00000u);
              s[m][u][e] = x;
              over = over || (x + (e & 1 ? lift[u].y : lift[u].x) > mx[m][e >> 1] + 8.f && ((see[m] >> (4 * u + e)) & 1));
            }
          if (__any_sync(0xffffffffu, over)) {
            // move the max of the rows to the largest score so far, rescale
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float top = mx[m][h];
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if ((see[m] >> (4 * u + 2 * h + e)) & 1) top = fmaxf(top, s[m][u][2 * h + e] + (e ? lift[u].y : lift[u].x));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
              const float f = top == mx[m][h] ? 1.f : exp2f(mx[m][h] - top);
              mx[m][h] = top;
              l[m][h] *= f;
#pragma unroll
              for (int j = 0; j < X::kTiles; ++j) {
                o[m][j][2 * h] *= f;
                o[m][j][2 * h + 1] *= f;
              }
            }
          }
        }
        // ---- weights ----
        uint32_t pr[kMT][4];
#pragma unroll
        for (int m = 0; m < kMT; ++m) {
          float e[2][4];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              float y = exp2_approx(s[m][u][x] - mx[m][x >> 1]);
              const bool seen = all || ((see[m] >> (4 * u + x)) & 1);
              y = seen ? y : 0.f;
              l[m][x >> 1] += y;
              if constexpr (k8) y = seen ? y * (x & 1 ? vs[u].y : vs[u].x) : 0.f;  // a hidden key's scale may be NaN
              e[u][x] = y;
            }
          pr[m][0] = pack<k8>(e[0][0], e[0][1]);
          pr[m][1] = pack<k8>(e[0][2], e[0][3]);
          pr[m][2] = pack<k8>(e[1][0], e[1][1]);
          pr[m][3] = pack<k8>(e[1][2], e[1][3]);
        }
        // ---- values ----
#pragma unroll
        for (int c = 0; c < X::kVC; ++c) {
          uint32_t vw[4][X::kVB / 4];
#pragma unroll
          for (int u = 0; u < 4; ++u) load_words<X::kVB / 4>(ring_v + from + (u * X::kVC + c) * 32 * X::kVB, vw[u]);
#pragma unroll
          for (int x = 0; x < X::kVB / 4; ++x) {
            if constexpr (k8) {
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const uint32_t b0 = join_codes<kMode>(vw[0][x], vw[1][x], y), b1 = join_codes<kMode>(vw[2][x], vw[3][x], y);
#pragma unroll
                for (int m = 0; m < kMT; ++m) mma<true>(o[m][4 * x + y], pr[m], b0, b1);
              }
            } else {
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t b0 = __byte_perm(vw[0][x], vw[1][x], y ? 0x7632 : 0x5410);
                const uint32_t b1 = __byte_perm(vw[2][x], vw[3][x], y ? 0x7632 : 0x5410);
#pragma unroll
                for (int m = 0; m < kMT; ++m) mma<false>(o[m][8 * c + 2 * x + y], pr[m], b0, b1);
              }
            }
          }
        }
      }

      // ---- the piece is done: warps together, two rows at a time ----
#pragma unroll
      for (int m = 0; m < kMT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 1);
          l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 2);
          if (t == 0) {
            sm.m[warp][16 * m + 8 * h + g] = mx[m][h];
            sm.l[warp][16 * m + 8 * h + g] = l[m][h];
          }
        }
      __syncthreads();
      const int64_t rows_left = p.q.T * p.group - (int64_t)rt * kRows;
      const int rows = rows_left < kRows ? (int)rows_left : kRows;
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 2) {
        // this lane's row, when it is one of the two
        const int m_of = r0 >> 4, h_of = (r0 >> 3) & 1;
        if ((g & ~1) == (r0 & 7)) {
          const int r = (r0 & ~7) + g;
          float top = -INFINITY;
          for (int x = 0; x < NW; ++x) top = fmaxf(top, sm.m[x][r]);
          const float own = sm.m[warp][r];
          // a warp that saw no key of the row has nothing to add
          const float f = sm.l[warp][r] == 0.f ? 0.f : own == top ? 1.f : exp2f(own - top);
          float* dst = sm.sum + (warp * 2 + (g & 1)) * kD;
#pragma unroll
          for (int m = 0; m < kMT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (m == m_of && h == h_of) {
#pragma unroll
                for (int j = 0; j < X::kTiles; ++j) {
                  const int d0 = k8 ? X::kVB * 2 * t + j : (j >> 3) * 64 + 16 * t + (j & 7);
                  const int d1 = d0 + (k8 ? X::kVB : 8);
                  dst[d0] = f == 0.f ? 0.f : f * o[m][j][2 * h];
                  dst[d1] = f == 0.f ? 0.f : f * o[m][j][2 * h + 1];
                }
              }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * kD; i += X::kThreads) {
          const int r = r0 + i / kD, col = i % kD;
          float top = -INFINITY, sum = 0.f, acc = 0.f;
          for (int x = 0; x < NW; ++x) top = fmaxf(top, sm.m[x][r]);
          for (int x = 0; x < NW; ++x) {
            const float lx = sm.l[x][r];
            if (lx != 0.f) sum = fmaf(sm.m[x][r] == top ? 1.f : exp2f(sm.m[x][r] - top), lx, sum);
            acc += sm.sum[x * 2 * kD + i];
          }
          // -kMost: nothing but biases of the type's lowest value
          const float m = top == -kMost ? -kMost : top * kLn2;
          const TreeRow row = tree_row(p, w.hk, rt, r);
          if (r >= rows) continue;
          if (row.t >= w.s.cnt) sum = 0.f;  // a row that does not exist
          if (w.part >= 0) {
            const int64_t part = p.part_row(span, rt, w.part, r);
            if (col < d) p.part_o[part * kTreePartCols + col] = acc;
            if (col == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m, sum);
          } else {
            if (col < d) tree_out_row<__nv_bfloat16>(p, w.b, row)[col] = __float2bfloat16_rn(sum != 0.f ? acc / sum : 0.f);
            if (col == 0 && p.q.lse)
              p.q.lse[((int64_t)w.b * p.q.n_q_heads + row.h) * p.q.T + row.t] = sum != 0.f ? m + logf(sum) : -INFINITY;
          }
        }
        __syncthreads();
      }
      base += w.k1 - w.k0;
    }
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");
}

template <int kMode, int kD, int kMT>
static int launch(const TreeParams& p, cudaStream_t st) {
  using X = Shape<kMode, kD, kMT>;
  constexpr size_t smem = sizeof(Smem<X, kMT>);
  static_assert(smem <= kSmemLimit, "shared memory");
  auto kernel = tree_mma_kernel<kMode, kD, kMT>;
  DCC_CHECK(check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "tree_mma smem"));
  kernel<<<p.n_groups * p.n_spans, X::kThreads, smem, st>>>(p);
  return check_launch("tree_attention");
}
template <int kMode>
static int launch_d(const TreeParams& p, cudaStream_t st) {
  if (p.c.head_dim <= 64) return p.n_rows == 16 ? launch<kMode, 64, 1>(p, st) : launch<kMode, 64, 2>(p, st);
  return p.n_rows == 16 ? launch<kMode, 128, 1>(p, st) : launch<kMode, 128, 2>(p, st);
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
