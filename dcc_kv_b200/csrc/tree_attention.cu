// Attention of the newest tokens over the paged cache: the C entry point, the
// CUDA-core kernel for every type and size, and the merge of partial results.
#include <algorithm>
#include <string>

#include "tree_attention.cuh"

namespace dcc {

constexpr int kSimtRows = 8;
constexpr int kSimtThreads = 128;  // one key of a tile, or one column of the head, per thread
constexpr int kSimtCtasPerSm = 6;

// Online softmax over key tiles of 128: thread = key for the scores (q rows
// from shared memory), thread = column for the values.  fp32 throughout.
// Bound by its loads of keys: a warp's 32 lanes read single elements a row apart,
// so that 2/3 of the time is waiting for them (19 % of the issue slots are used).
// It serves fp32 queries and caches and the head_dims and page sizes that the
// tensor-core kernels do not take.  16 sequences, 4 heads on each of 8 KV heads
// of 128, 8k tokens: 1110 us beside a bf16 cache whose pages hold 12 tokens or
// one, where 16-token pages take tree_mma.cu 102 us; 1165 us beside fp32.
template <typename T, int kFormat>
__global__ void __launch_bounds__(kSimtThreads) tree_simt_kernel(const __grid_constant__ TreeParams p) {
  constexpr bool kScaled = kFormat == DCC_KV_INT8 || kFormat == DCC_KV_E4M3;
  __shared__ TreePlanSmem ps;
  __shared__ __align__(16) float q_s[128][kSimtRows];  // [column][row]
  __shared__ __align__(16) float x_s[kTreeKeys][kSimtRows];  // scores, then probabilities (-0: not seen)
  __shared__ float m_s[kSimtRows], l_s[kSimtRows], corr_s[kSimtRows];
  __shared__ int64_t row_s[kTreeKeys];  // cache row of each key, -1: none
  __shared__ float vscale_s[kTreeKeys];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int d = p.c.head_dim;
  const int span = blockIdx.x / p.n_groups;
  tree_plan(p, span, ps);
  for (int rt = blockIdx.x % p.n_groups; rt < p.n_row_tiles; rt += p.n_groups) {
    TreeWalk walk;
    walk.start(p, ps.plan);
    TreePiece w;
    while (walk.next(p, w)) {
      __syncthreads();
      if (tid < kSimtRows) {
        m_s[tid] = -INFINITY;
        l_s[tid] = 0.f;
      }
      for (int i = tid; i < kSimtRows * d; i += kSimtThreads) {
        const int r = i / d, c = i - r * d;
        const TreeRow row = tree_row(p, w.hk, rt, r);
        q_s[c][r] = row.exists ? to_f32<T>(static_cast<const T*>(p.q.q)[w.b * p.q.q_seq_stride + row.h * p.q.q_head_stride +
                                                                        row.t * p.q.q_row_stride + c])
                               : 0.f;
      }
      float o[kSimtRows];
#pragma unroll
      for (int r = 0; r < kSimtRows; ++r) o[r] = 0.f;
      const PageWalk pages{p.q.page_table + w.b * p.q.table_stride, p.c.n_pages, p.c.page_size, p.q.max_pages};
      for (int kt = w.k0; kt < w.k1; ++kt) {
        __syncthreads();
        {
          const int64_t pos = (int64_t)kt * kTreeKeys + tid;
          int off = 0;
          const int64_t page = pos < w.s.total ? pages.page_of(pos, off) : -1;
          const int64_t at = page >= 0 ? page_row(p.c, page, w.hk, off) : -1;
          row_s[tid] = at;
          float x[kSimtRows];
#pragma unroll
          for (int r = 0; r < kSimtRows; ++r) x[r] = 0.f;
          float bias = 0.f, ks = 1.f;
          if (at >= 0) {
            for (int c = 0; c < d; ++c) {
              const float kv = load_code<kFormat>(p.c.k, at * d + c);
#pragma unroll
              for (int r = 0; r < kSimtRows; ++r) x[r] = fmaf(q_s[c][r], kv, x[r]);
            }
            if (p.c.bias) bias = p.c.bias[at];
            if (kScaled) {
              ks = p.c.k_scale[at];
              vscale_s[tid] = p.c.v_scale[at];
            }
          }
          const int64_t i = pos - w.s.ctx;  // >= 0: newest token i
#pragma unroll
          for (int r = 0; r < kSimtRows; ++r) {
            const TreeRow row = tree_row(p, w.hk, rt, r);
            const bool sees = at >= 0 && row.exists && row.t < w.s.cnt && (i < 0 || tree_sees(p, w.b, row.t, i));
            x_s[tid][r] = sees ? fmaf(x[r] * ks, p.scale, bias) : __uint_as_float(0xffffffffu);  // mark: not seen
          }
        }
        __syncthreads();
        // rows 2 warp, 2 warp + 1
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const int r = 2 * warp + rr;
          float x[4], mt = -INFINITY;
          bool seen[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = x_s[lane + 32 * i][r];
            seen[i] = __float_as_uint(x[i]) != 0xffffffffu;
            if (seen[i]) mt = fmaxf(mt, x[i]);
          }
          const float m_old = m_s[r];
          const float m_new = fmaxf(m_old, warp_max(mt));
          const float msub = m_new == -INFINITY ? 0.f : m_new;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = seen[i] ? expf(x[i] - msub) : 0.f;
            sum += e;
            float pv = e;
            if (kScaled && seen[i]) pv *= vscale_s[lane + 32 * i];
            x_s[lane + 32 * i][r] = seen[i] ? pv : -0.f;
          }
          sum = warp_sum(sum);
          if (lane == 0) {
            const float corr = m_old == -INFINITY ? 0.f : expf(m_old - m_new);
            m_s[r] = m_new;
            l_s[r] = l_s[r] * corr + sum;
            corr_s[r] = corr;
          }
        }
        __syncthreads();
        if (tid < d) {
#pragma unroll
          for (int r = 0; r < kSimtRows; ++r) o[r] *= corr_s[r];
          const int64_t left = w.s.total - (int64_t)kt * kTreeKeys;
          const int n = left < kTreeKeys ? (int)left : kTreeKeys;
#pragma unroll 4
          for (int j = 0; j < n; ++j) {
            const int64_t at = row_s[j];
            if (at < 0) continue;
            const float vv = load_code<kFormat>(p.c.v, at * d + tid);
#pragma unroll
            for (int r = 0; r < kSimtRows; ++r) {
              const float pr = x_s[j][r];
              if (__float_as_uint(pr) != 0x80000000u) o[r] = fmaf(pr, vv, o[r]);  // nothing of a key that is not seen
            }
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kSimtRows; ++r) {
        if (w.part >= 0) {
          const int64_t slot = p.part_row(span, rt, w.part, r);
          if (tid < d) p.part_o[slot * kTreePartCols + tid] = l_s[r] == 0.f ? 0.f : o[r] / l_s[r];
          if (tid == 0) {
            p.part_ml[slot * 2] = m_s[r];
            p.part_ml[slot * 2 + 1] = l_s[r];
          }
        } else {
          const TreeRow row = tree_row(p, w.hk, rt, r);
          if (!row.exists) continue;
          const float l = l_s[r];
          if (tid < d) tree_out_row<T>(p, w.b, row)[tid] = from_f32<T>(l == 0.f ? 0.f : o[r] / l);
          if (tid == 0 && p.q.lse)
            p.q.lse[((int64_t)w.b * p.q.n_q_heads + row.h) * p.q.T + row.t] = l == 0.f ? -INFINITY : m_s[r] + logf(l);
        }
      }
    }
  }
}

constexpr int kMergeWarps = 4;

// One warp per row of an item that several CTAs worked on (or that no key
// tile belongs to): with w_i = e^(m_i - m) l_i, o = sum_i w_i O_i / sum_i w_i
// (O_i is an output already, so whatever the sizes of the values are, only
// weights are compared here).
template <typename T>
__global__ void __launch_bounds__(kMergeWarps * 32) tree_merge_kernel(const __grid_constant__ TreeParams p) {
  __shared__ int64_t sums[2][kMergeWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t items = (int64_t)p.c.n_kv_heads * p.n_row_tiles;
  const int b = (int)(blockIdx.x / items);
  const int item = (int)(blockIdx.x - b * items);
  const int hk = item / p.n_row_tiles, rt = item - hk * p.n_row_tiles;
  int64_t before = 0, all = 0;
  for (int i = threadIdx.x; i < p.q.n_seqs; i += kMergeWarps * 32) {
    const int64_t w = p.c.n_kv_heads * tree_key_tiles(tree_tokens(p, i));
    all += w;
    if (i < b) before += w;
  }
  before = warp_sum(before);
  all = warp_sum(all);
  if (lane == 0) {
    sums[0][warp] = before;
    sums[1][warp] = all;
  }
  __syncthreads();
  before = all = 0;
  for (int i = 0; i < kMergeWarps; ++i) {
    before += sums[0][i];
    all += sums[1][i];
  }
  const SeqTokens s = tree_tokens(p, b);
  const int64_t tiles = tree_key_tiles(s), first = before + hk * tiles;
  int i0 = 0, i1 = -1;
  if (tiles > 0) {
    const int n = span_count(all, p.n_spans);
    i0 = span_owner(all, first, n);
    i1 = span_owner(all, first + tiles - 1, n);
    if (i0 == i1) return;
  }
  const int r = blockIdx.y * kMergeWarps + warp;
  if (r >= p.n_rows) return;
  const TreeRow row = tree_row(p, hk, rt, r);
  if (!row.exists) return;
  auto slot = [&](int i) { return p.part_row(i, rt, i == i0 ? 1 : 0, r); };
  float m = -INFINITY;
  for (int i = i0 + lane; i <= i1; i += 32) m = fmaxf(m, p.part_ml[slot(i) * 2]);
  m = warp_max(m);
  const float msub = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = i0; i <= i1; ++i) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot(i) * 2);
    const float4 v = *reinterpret_cast<const float4*>(p.part_o + slot(i) * kTreePartCols + lane * 4);
    if (ml.y == 0.f) continue;  // no key of that part was seen; its O holds nothing
    const float w = expf(ml.x - msub) * ml.y;
    l += w;
    o[0] = fmaf(w, v.x, o[0]);
    o[1] = fmaf(w, v.y, o[1]);
    o[2] = fmaf(w, v.z, o[2]);
    o[3] = fmaf(w, v.w, o[3]);
  }
  const int d = p.c.head_dim;
  T* out = tree_out_row<T>(p, b, row);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane * 4 + c < d) out[lane * 4 + c] = from_f32<T>(l == 0.f ? 0.f : o[c] / l);
  if (lane == 0 && p.q.lse)
    p.q.lse[((int64_t)b * p.q.n_q_heads + row.h) * p.q.T + row.t] =
        l == 0.f ? -INFINITY : m + logf(l);
}

bool tree_tensor_supported(const dcc_kv_pages& c, const dcc_tree_query& q, int dtype) {
  // rows of 16-byte chunks, eight rows that never leave their page
  // (a pool without pages is nothing to make a tensor map of)
  if (dtype != DCC_BF16 || c.format == DCC_KV_F32 || c.head_dim % 16 != 0 || c.page_size % 8 != 0 || c.n_pages == 0) return false;
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

// Which kernel takes a call, with how many query rows per KV head at a time.
// Up to 16 rows the warps of tree_mma.cu, which pay per 8 rows, are ahead of
// the tensor core tiles of tree_tc05.cu, which pay for 128 or 256 whatever the
// number is (beside 16 bf16 rows they are level); above they are behind (16
// sequences, 8 KV heads of 128, us):
//   rows  tokens  int8 mma / tc05   bf16 mma / tc05
//      8    8192       82 / 159         107 / 115
//     16    8192      112 / 160         116 / 114
//     32    4096      125 / 98          117 / 74
//     32     512      175 / 98          183 / 90    (64 sequences)
// Within them 8 rows at a time where that is all (one token of 16 sequences over
// 8192, int8: 75 us, in 16 rows 92); one tile of 128 rows up to 128 (52 rows, 16
// sequences of 4001 int8 tokens: 104 us, as a pair 138); beyond, beside 8-bit
// codes, pairs of them that share each key tile and its widening (256 rows over
// 131072 tokens, int8: 290 us, one by one 320).  bf16 tiles, with nothing to widen,
// come to CTAs side by side from the L2 as well (256 rows over 131072 tokens 193 us,
// as pairs 200; over 8 sequences of 8192 126, 138; over 64 of 512 208, 199).
// What neither takes (other types, odd strides or sizes) goes to the plain
// kernel of this file.
enum class Path { kSimt, kMma, kTc05 };
constexpr int kMmaRows = 16;

static Path tree_params(const dcc_kv_pages& c, const dcc_tree_query& q, int dtype, TreeParams& p) {
  p.c = c;
  p.q = q;
  p.group = q.n_q_heads / c.n_kv_heads;
  const int64_t rows = q.T * p.group;
  const Path path = !tree_tensor_supported(c, q, dtype) ? Path::kSimt : rows <= kMmaRows ? Path::kMma : Path::kTc05;
  p.n_rows = path == Path::kSimt ? kSimtRows : rows <= 8 ? 8 : rows <= kMmaRows ? kMmaRows
             : rows <= 128 || c.format == DCC_KV_BF16 ? 128 : 256;
  p.n_row_tiles = (int)((rows + p.n_rows - 1) / p.n_rows);
  const int ctas = num_sms() * (path == Path::kSimt ? kSimtCtasPerSm : 1);
  const int rounds = (p.n_row_tiles + ctas - 1) / ctas;
  p.n_groups = rounds > 0 ? (p.n_row_tiles + rounds - 1) / rounds : 1;
  p.n_spans = ctas / p.n_groups;
  return path;
}

static size_t tree_carve(TreeParams& p, Workspace& ws) {
  const size_t slots = p.n_spans > 1 ? (size_t)p.part_row(p.n_spans, 0, 0, 0) : 0;  // one span leaves no parts
  p.part_o = ws.take<float>(slots * kTreePartCols);
  p.part_ml = ws.take<float>(slots * 2);
  return align_up(ws.used, 256);
}

static int tree_check(const dcc_kv_pages* cache, const dcc_tree_query* q, int dtype) {
  DCC_CHECK(check_pages(cache, "tree_attention"));
  if (!q || q->T < 0 || q->n_seqs < 0 || q->max_pages < 0 || q->n_q_heads < 1)
    return fail(DCC_ERR_INVALID_ARGUMENT, "tree_attention: bad query");
  if (q->n_q_heads % cache->n_kv_heads)
    return fail(DCC_ERR_INVALID_ARGUMENT, "tree_attention: n_q_heads must be a multiple of n_kv_heads");
  if (dtype != DCC_F32 && dtype != DCC_BF16) return fail(DCC_ERR_DTYPE, "tree_attention: unsupported dtype");
  if (q->T > kTreeMaxT) return fail(DCC_ERR_UNSUPPORTED, "tree_attention: at most 4096 newest tokens");
  if (q->T * q->n_q_heads > (1 << 24)) return fail(DCC_ERR_UNSUPPORTED, "tree_attention: too many query rows");
  return DCC_OK;
}

template <typename T>
static void tree_simt_launch(const TreeParams& p, cudaStream_t st) {
  switch (p.c.format) {
    case DCC_KV_BF16: tree_simt_kernel<T, DCC_KV_BF16><<<p.n_groups * p.n_spans, kSimtThreads, 0, st>>>(p); break;
    case DCC_KV_F32: tree_simt_kernel<T, DCC_KV_F32><<<p.n_groups * p.n_spans, kSimtThreads, 0, st>>>(p); break;
    case DCC_KV_INT8: tree_simt_kernel<T, DCC_KV_INT8><<<p.n_groups * p.n_spans, kSimtThreads, 0, st>>>(p); break;
    default: tree_simt_kernel<T, DCC_KV_E4M3><<<p.n_groups * p.n_spans, kSimtThreads, 0, st>>>(p); break;
  }
}

}  // namespace dcc

using namespace dcc;

extern "C" size_t dcc_tree_attention_workspace_bytes(const dcc_kv_pages* cache, const dcc_tree_query* query, int dtype) {
  if (tree_check(cache, query, dtype) != DCC_OK) return 0;
  TreeParams p{};
  tree_params(*cache, *query, dtype, p);
  Workspace ws(nullptr, 0);
  return tree_carve(p, ws);
}

extern "C" int dcc_tree_attention(const dcc_kv_pages* cache, const dcc_tree_query* query, double scale, int dtype,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  DCC_CHECK(tree_check(cache, query, dtype));
  const dcc_tree_query& q = *query;
  if (q.T == 0 || q.n_seqs == 0) return DCC_OK;
  if (!q.q || !q.o || !q.context || (q.max_pages > 0 && !q.page_table))
    return fail(DCC_ERR_INVALID_ARGUMENT, "tree_attention: null tensor");
  TreeParams p{};
  const Path path = tree_params(*cache, q, dtype, p);
  p.scale = (float)scale;
  Workspace ws(workspace, workspace_bytes);
  tree_carve(p, ws);
  if (!workspace || !ws.ok()) return fail(DCC_ERR_WORKSPACE, "tree_attention: workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) & 15u)  // the parts are stored and read 16 bytes at a time
    return fail(DCC_ERR_INVALID_ARGUMENT, "tree_attention: the workspace must be 16-byte aligned");
  const int64_t items = (int64_t)q.n_seqs * cache->n_kv_heads * p.n_row_tiles;
  if (items > 2147483647LL) return fail(DCC_ERR_UNSUPPORTED, "tree_attention: too many sequences");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (path == Path::kMma) {
    DCC_CHECK(launch_tree_mma(p, st));
  } else if (path == Path::kTc05) {
    DCC_CHECK(launch_tree_tc05(p, st));
  } else {
    if (dtype == DCC_BF16) tree_simt_launch<__nv_bfloat16>(p, st);
    else tree_simt_launch<float>(p, st);
    DCC_CHECK(check_launch("tree_attention"));
  }
  const int rows = (int)std::min<int64_t>(p.n_rows, q.T * p.group);
  const dim3 grid((unsigned)items, (unsigned)((rows + kMergeWarps - 1) / kMergeWarps));
  if (dtype == DCC_BF16) tree_merge_kernel<__nv_bfloat16><<<grid, kMergeWarps * 32, 0, st>>>(p);
  else tree_merge_kernel<float><<<grid, kMergeWarps * 32, 0, st>>>(p);
  return check_launch("tree_attention merge");
}
