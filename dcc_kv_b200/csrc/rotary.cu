// Rotary positions of queries and keys in one launch.
//
// A thread owns one chunk of V pairs of one token and walks over heads: the
// V sines and cosines (the only real arithmetic) are computed once and used
// for every head of the thread, so the kernel is bound by memory.  Angles are
// formed in turns (position * turns_per_position, fp64) and reduced to
// [-1/2, 1/2] turn before the fp32 sine and cosine: at position 2^20 an fp32
// angle would be off by 0.06 rad, this one by 2e-7.
// Measured: 32 + 8 heads of 128 in bf16, 32768 tokens, 112 us or 6.0 TB/s, with the
// gradient 221; 2 x 4097 tokens with the gradient, in a graph, fp32 112 us or 6.0 TB/s,
// bf16 68 or 5.0 (as calls 145 to 150, which is the host's part of autograd).  Rows that are
// not 16-byte aligned, 20 heads of 32768 tokens: bf16 135 us (aligned 66), fp32 147
// (118), fp64 220 (212).  A single token of 64 sequences takes 3 us in a graph, 21
// with the Python call.
#include <algorithm>
#include <string>

#include "common.cuh"

namespace dcc {

constexpr int kMaxFreqs = 128;
constexpr int kRotThreads = 256;

struct RotaryParams {
  dcc_rotary_tensor t[2];
  int n_heads;         // of both tensors together
  int heads_per_thread;
  const void* pos;
  int64_t pos_seq_stride, pos_row_stride;
  int pos64;
  int64_t n_seqs, T;
  int d, n_freqs;
  int n_rot, n_chunks;  // chunks of a head: n_rot of V pairs each, then copies of 2 V elements
  float sign;
  double magnitude;
  double turns[kMaxFreqs];
};

// V consecutive elements; V * sizeof(T) is 16, 32 or 64 bytes, or one element.
template <typename T, int V>
struct alignas(V * sizeof(T) >= 16 ? 16 : sizeof(T)) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ void load_pack(Pack<T, V>& p, const T* src) {
  if constexpr (V == 1) {
    p.v[0] = *src;
  } else {
    static_assert((V * sizeof(T)) % 16 == 0, "16-byte packs");
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(p.v)[i] = reinterpret_cast<const uint4*>(src)[i];
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* dst, const Pack<T, V>& p) {
  if constexpr (V == 1) {
    *dst = p.v[0];
  } else {
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(p.v)[i];
  }
}

template <typename T> struct RotAcc { using type = float; };
template <> struct RotAcc<double> { using type = double; };

__device__ __forceinline__ void sincos_turns(double turns, float& s, float& c) {
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
}
__device__ __forceinline__ void sincos_turns(double turns, double& s, double& c) {
  sincospi(2.0 * (turns - rint(turns)), &s, &c);
}

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  using A = typename RotAcc<T>::type;
  const int64_t per_head_group = p.n_seqs * p.T * p.n_chunks;
  const int64_t id = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  if (id >= per_head_group) return;
  const int c = (int)(id % p.n_chunks);
  const int64_t row = id / p.n_chunks;
  const int64_t b = row / p.T, t = row - b * p.T;
  const int h0 = blockIdx.y * p.heads_per_thread;
  const int h1 = min(h0 + p.heads_per_thread, p.n_heads);
  const int nh0 = (int)p.t[0].n_heads;
  const bool rot = c < p.n_rot;
  // offsets of the two packs in the head
  int o1, o2;
  if (!rot) {
    o1 = 2 * p.n_freqs + (c - p.n_rot) * 2 * V;
    o2 = o1 + V;
  } else if (kInterleaved) {
    o1 = c * 2 * V;
    o2 = o1 + V;
  } else {
    o1 = c * V;
    o2 = o1 + p.n_freqs;
  }
  const bool two = rot || o2 < p.d;  // the copied tail may end with a single pack
  A sn[V], cs[V];
  if (rot) {
    const int64_t at = b * p.pos_seq_stride + t * p.pos_row_stride;
    const double pos = p.pos64 ? (double)static_cast<const int64_t*>(p.pos)[at]
                               : (double)static_cast<const int32_t*>(p.pos)[at];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sincos_turns(pos * p.turns[c * V + i], sn[i], cs[i]);
      sn[i] *= (A)p.magnitude * (A)p.sign;
      cs[i] *= (A)p.magnitude;
    }
  }
#pragma unroll 2
  for (int h = h0; h < h1; ++h) {
    const bool second = h >= nh0;
    const dcc_rotary_tensor& q = second ? p.t[1] : p.t[0];
    const int hh = second ? h - nh0 : h;
    const T* x = static_cast<const T*>(q.x) + b * q.x_seq_stride + hh * q.x_head_stride + t * q.x_row_stride;
    T* y = static_cast<T*>(q.y) + b * q.y_seq_stride + hh * q.y_head_stride + t * q.y_row_stride;
    Pack<T, V> a, z;
    load_pack<T, V>(a, x + o1);
    if (two) load_pack<T, V>(z, x + o2);
    if (rot) {
      if constexpr (kInterleaved) {
        T* e = a.v;
        T* f = z.v;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // pair i: elements 2i, 2i + 1 of the 2 V loaded ones
          T& l = 2 * i < V ? e[2 * i < V ? 2 * i : 0] : f[2 * i < V ? 0 : 2 * i - V];
          T& r = 2 * i + 1 < V ? e[2 * i + 1 < V ? 2 * i + 1 : 0] : f[2 * i + 1 < V ? 0 : 2 * i + 1 - V];
          const A u = to_acc<A, T>(l), w = to_acc<A, T>(r);
          l = (T)(u * cs[i] - w * sn[i]);
          r = (T)(u * sn[i] + w * cs[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const A u = to_acc<A, T>(a.v[i]), w = to_acc<A, T>(z.v[i]);
          a.v[i] = (T)(u * cs[i] - w * sn[i]);
          z.v[i] = (T)(u * sn[i] + w * cs[i]);
        }
      }
    }
    store_pack<T, V>(y + o1, a);
    if (two) store_pack<T, V>(y + o2, z);
  }
}

template <typename T, int V>
static int rotary_launch(RotaryParams& p, bool interleaved, cudaStream_t st) {
  p.n_rot = p.n_freqs / V;
  const int rest = p.d - 2 * p.n_freqs;
  p.n_chunks = p.n_rot + (rest / V + 1) / 2;
  const int64_t threads = p.n_seqs * p.T * p.n_chunks;
  // enough threads to fill the GPU twice; beyond that every further head of a
  // thread saves its sines and cosines
  const int64_t want = (int64_t)num_sms() * 2048 * 2;
  const int64_t groups = std::min<int64_t>(p.n_heads, std::max<int64_t>(1, (want + threads - 1) / threads));
  p.heads_per_thread = (int)((p.n_heads + groups - 1) / groups);
  const int64_t blocks = (threads + kRotThreads - 1) / kRotThreads;
  if (blocks > 2147483647LL) return fail(DCC_ERR_UNSUPPORTED, "rotary: too many tokens");
  const dim3 grid((unsigned)blocks, (unsigned)((p.n_heads + p.heads_per_thread - 1) / p.heads_per_thread));
  if (interleaved) rotary_kernel<T, V, true><<<grid, kRotThreads, 0, st>>>(p);
  else rotary_kernel<T, V, false><<<grid, kRotThreads, 0, st>>>(p);
  return check_launch("rotary");
}

template <typename T>
static int rotary_typed(RotaryParams& p, int n_tensors, bool interleaved, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // 16-byte packs where every pack starts on a 16-byte boundary
  bool wide = p.n_freqs % V == 0 && p.d % V == 0;
  for (int i = 0; i < n_tensors; ++i) {
    const dcc_rotary_tensor& q = p.t[i];
    wide = wide && ((reinterpret_cast<uintptr_t>(q.x) | reinterpret_cast<uintptr_t>(q.y)) & 15u) == 0;
    for (int64_t s : {q.x_seq_stride, q.x_head_stride, q.x_row_stride, q.y_seq_stride, q.y_head_stride, q.y_row_stride})
      wide = wide && s % V == 0;
  }
  return wide ? rotary_launch<T, V>(p, interleaved, st) : rotary_launch<T, 1>(p, interleaved, st);
}

}  // namespace dcc

using namespace dcc;

extern "C" int dcc_rotary(const dcc_rotary_tensor* tensors, int n_tensors, const void* positions,
                          int positions_are_int64, int64_t pos_seq_stride, int64_t pos_row_stride, int64_t n_seqs,
                          int64_t T, int head_dim, int n_freqs, const double* turns, double magnitude, int layout,
                          int inverse, int dtype, void* stream) {
  if (!tensors || n_tensors < 1 || n_tensors > 2 || n_seqs < 0 || T < 0 || !turns)
    return fail(DCC_ERR_INVALID_ARGUMENT, "rotary: bad arguments");
  if (layout != DCC_ROTARY_HALF && layout != DCC_ROTARY_INTERLEAVED)
    return fail(DCC_ERR_INVALID_ARGUMENT, "rotary: unknown layout");
  if (n_freqs < 1 || n_freqs > kMaxFreqs || 2 * n_freqs > head_dim)
    return fail(DCC_ERR_UNSUPPORTED, "rotary: between 1 and 128 pairs, within the head");
  RotaryParams p{};
  int64_t heads = 0;
  for (int i = 0; i < n_tensors; ++i) {
    if (tensors[i].n_heads < 0) return fail(DCC_ERR_INVALID_ARGUMENT, "rotary: bad head count");
    heads += tensors[i].n_heads;
    p.t[i] = tensors[i];
  }
  if (n_seqs == 0 || T == 0 || heads == 0) return DCC_OK;
  if (heads > 65535) return fail(DCC_ERR_UNSUPPORTED, "rotary: too many heads");
  if (!positions) return fail(DCC_ERR_INVALID_ARGUMENT, "rotary: null positions");
  for (int i = 0; i < n_tensors; ++i)
    if (tensors[i].n_heads > 0 && (!tensors[i].x || !tensors[i].y))
      return fail(DCC_ERR_INVALID_ARGUMENT, "rotary: null tensor");
  p.n_heads = (int)heads;
  p.pos = positions;
  p.pos64 = positions_are_int64 != 0;
  p.pos_seq_stride = pos_seq_stride;
  p.pos_row_stride = pos_row_stride;
  p.n_seqs = n_seqs;
  p.T = T;
  p.d = head_dim;
  p.n_freqs = n_freqs;
  p.sign = inverse ? -1.f : 1.f;
  p.magnitude = magnitude;
  for (int i = 0; i < n_freqs; ++i) p.turns[i] = turns[i];
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool il = layout == DCC_ROTARY_INTERLEAVED;
  if (dtype == DCC_BF16) return rotary_typed<__nv_bfloat16>(p, n_tensors, il, st);
  if (dtype == DCC_F32) return rotary_typed<float>(p, n_tensors, il, st);
  if (dtype == DCC_F64) return rotary_typed<double>(p, n_tensors, il, st);
  return fail(DCC_ERR_DTYPE, "rotary: unsupported dtype");
}
